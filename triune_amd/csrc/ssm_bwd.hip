// ssm_bwd.hip -- gradients of the selective scan (dense calls) on gfx950.
//
// With gy = dy silu(z) and dh_t = C_t gy_t + a_{t+1} dh_{t+1}, a_t = exp(dt_t A):
//     dC_t,n = sum_d gy h          dB_t,n = sum_d dh dt u        p = dh a h_{t-1}
//     ddt = sum_n (p A + dh B u)   du = dt sum_n dh B + D gy     dA = sum_t p dt
//     ddelta = ddt softplus'(x)    dz = dy silu'(z) (sum_n C h + D u)
//
// Lanes, waves and tiles are those of the forward (ssm.hip).  The forward kept a state for each tile; a
// workgroup walks its tiles from the last to the first.  In a tile it runs the states forward once to
// have the one that each walk of eight tokens starts from, then takes the walks backward: a walk's decays
// and states are formed again and stay in registers (64 of them), so nothing of size tokens x channels x
// states goes to memory.  Sums over states (for dt, u, z) meet in LDS; sums over channels (dB, dC) are
// taken across the lanes, eight values of a token together by halving exchanges (fp32 matrix products
// with columns of the identity, which add four lanes, took 179 cycles per wave and state alone), and
// stored per workgroup; a last kernel adds the workgroups' parts in a fixed order, so the gradients do
// not depend on timing.
//
// Bound by vector issue at two waves a SIMD: 25 vector operations and 1.75 exp2 per wave and state (about
// 105 cycles).  4 x 2048 tokens of 1536 channels, N = 16, bf16: 206 us where that is 134.
#include "ssm.h"

namespace triune {

// Segmented calls: the gradient that reaches each segment's start from its own tokens,
// e <- a_t (C_t gy_t + e) from zero at its end, and the segment's sum of dt.  Laid out as ssm_scan_kernel.
template <typename T, int NW, int V>
__global__ __launch_bounds__(64 * NW) void ssm_bwd_states_kernel(SsmBwdParams g) {
    const SsmParams& a = g.f;
    constexpr int NS = 4, NT = 64 * NW, TT = NW == 1 || NW == 16 ? 16 : 32, LPR = 64 / V, TS = NT / LPR;
    constexpr int K = (TT + TS - 1) / TS, KB = TT * 4 * NW / NT, U = 2, ES = sizeof(T);
    __shared__ __attribute__((aligned(16))) float s_d[2][TT][64];  // dt, gy
    __shared__ __attribute__((aligned(16))) float s_c[TT][NW][NS];

    const int nblk = a.G * a.blocks;
    const int64_t work = blockIdx.x / nblk;
    const int cb = (int)(blockIdx.x - work * nblk);
    SsmSeg sg;
    ssm_segment(a, work, sg);
    const int Dg = a.Dm / a.G, grp = cb / a.blocks, c0 = (cb - grp * a.blocks) * 64;
    const int lane = threadIdx.x & 63, w = wave_index(), n0 = NS * w;
    const bool chv = c0 + lane < Dg;
    const int ch = grp * Dg + (chv ? c0 + lane : 0);
    const int cl = (threadIdx.x % LPR) * V, tl = threadIdx.x / LPR;
    const bool lv = c0 + cl < Dg && (TS <= TT || tl < TT);
    const int lch = grp * Dg + (lv ? c0 + cl : 0);
    const int bn = threadIdx.x % (4 * NW), bt = threadIdx.x / (4 * NW);
    const T* pd = (const T*)a.dl.p + sg.seq * a.dl.sb + sg.t0 * a.dl.st;
    const T* pz = a.z.p ? (const T*)a.z.p + sg.seq * a.z.sb + sg.t0 * a.z.st : nullptr;
    const T* py = (const T*)g.dy.p + sg.seq * g.dy.sb + sg.t0 * g.dy.st;
    const T* pC = (const T*)a.C + sg.seq * a.c_sb + sg.t0 * a.c_st + grp * a.c_sg;
    float Al[NS], e[NS], bias[V], sum[V];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        Al[j] = n0 + j < a.N ? log2_decay(a.A[(int64_t)ch * a.N + n0 + j]) : 0.f;
        e[j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) bias[j] = a.bias ? a.bias[lch + j] : 0.f, sum[j] = 0.f;
    Vec<T, V> rd[K], rz[K], ry[K];
    Vec<T, 1> rc[KB];
    const int vd = lv ? (tl * (int)a.dl.st + lch) * ES : TILE_SKIP, vz = lv ? (tl * (int)a.z.st + lch) * ES : TILE_SKIP;
    const int vy = lv ? (tl * (int)g.dy.st + lch) * ES : TILE_SKIP;
    const int vc = bn < a.N ? (bt * (int)a.c_st + bn) * ES : TILE_SKIP;
    auto fetch = [&](int t0) {
        const int left = t0 < 0 ? 0 : sg.len - t0;
        tile_load_rows(tile_rows(pd + t0 * a.dl.st, a.dl.st, left, a.Dm), vd, TS * ES * (int)a.dl.st, rd);
        tile_load_rows(tile_rows(py + t0 * g.dy.st, g.dy.st, left, a.Dm), vy, TS * ES * (int)g.dy.st, ry);
        tile_load_rows(tile_rows(pz ? pz + t0 * a.z.st : pz, a.z.st, left, a.Dm), vz, TS * ES * (int)a.z.st, rz);
        tile_load_rows(tile_rows(pC + t0 * a.c_st, a.c_st, left, a.N), vc, 16 * ES * (int)a.c_st, rc);
    };
    struct Block {
        float dt[U], gy[U], c[U][NS];
    };
    auto read = [&](Block& x, int t) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            x.dt[i] = s_d[0][t + i][lane];
            x.gy[i] = s_d[1][t + i][lane];
#pragma unroll
            for (int j = 0; j < NS; ++j) x.c[i][j] = s_c[t + i][w][j];
        }
    };
    auto walk = [&](const Block& x) {
#pragma unroll
        for (int i = U - 1; i >= 0; --i)
#pragma unroll
            for (int j = 0; j < NS; ++j)
                e[j] = __builtin_amdgcn_exp2f(x.dt[i] * Al[j]) * __builtin_fmaf(x.c[i][j], x.gy[i], e[j]);
    };
    const int tiles = (sg.len + TT - 1) / TT;
    fetch((tiles - 1) * TT);
    for (int k = tiles - 1; k >= 0; --k) {
        const int t0 = k * TT;
        float dt[K][V], gy[K][V];
#pragma unroll
        for (int i = 0; i < K; ++i) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float x = (float)rd[i].v[j] + bias[j], y = (float)ry[i].v[j];
                dt[i][j] = a.softplus ? softplus(x) : x;
                gy[i][j] = pz ? y * silu_gate((float)rz[i].v[j]) : y;
            }
            if (t0 + i * TS + tl >= sg.len) {
#pragma unroll
                for (int j = 0; j < V; ++j) dt[i][j] = gy[i][j] = 0.f;
            }
            if (TS <= TT || tl < TT) {
                lds_store<V>(&s_d[0][i * TS + tl][cl], dt[i]);
                lds_store<V>(&s_d[1][i * TS + tl][cl], gy[i]);
#pragma unroll
                for (int j = 0; j < V; ++j) sum[j] += dt[i][j];
            }
        }
#pragma unroll
        for (int i = 0; i < KB; ++i) s_c[i * 16 + bt][bn >> 2][bn & 3] = t0 + i * 16 + bt < sg.len ? (float)rc[i].v[0] : 0.f;
        fetch(t0 - TT);
        __syncthreads();
        if (n0 < a.N) {
            Block p, q;
            read(p, TT - U);
#pragma unroll 1
            for (int t = TT - 2 * U; t >= 0; t -= 2 * U) {
                read(q, t);
                walk(p);
                read(p, t >= U ? t - U : 0);
                walk(q);
            }
        }
        __syncthreads();
    }
    if (chv) {
#pragma unroll
        for (int j = 0; j < NS; ++j)
            if (n0 + j < a.N) a.ws_state[(work * a.N + n0 + j) * a.Dm + ch] = e[j];
    }
    if (TS <= TT || tl < TT) lds_store<V>(&s_d[0][tl][cl], sum);
    __syncthreads();
    if (w == 0 && chv) {
        float s = 0.f;
        for (int k = 0; k < (TS < TT ? TS : TT); ++k) s += s_d[0][k][lane];
        a.ws_sum[work * a.Dm + ch] = s;
    }
}

// The sums over a wave's lanes of v[0..8), by halving exchanges: a level leaves half of the values to each
// half of the lanes.  Lane l holds the one of value l / 8.
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

// Operands in LDS are read again by each phase and for each pair of tokens: kept from one to the next
// they would take a hundred registers.
__device__ __forceinline__ void reread() { asm volatile("" ::: "memory"); }

template <typename T, int NW, int V>
__global__ __launch_bounds__(64 * NW, NW == 16 ? 4 : NW == 1 ? 1 : 2) void ssm_bwd_kernel(SsmBwdParams g) {
    const SsmParams& a = g.f;
    constexpr int NS = 4, NT = 64 * NW, TT = NW == 16 ? 16 : 32, LPR = 64 / V, TS = NT / LPR;  // TT: ssm_kept_every
    constexpr int K = (TT + TS - 1) / TS, KB = TT * 4 * NW / NT, ES = sizeof(T);
    constexpr int SB = NW <= 4 ? 16 : NW == 8 ? 8 : 4;  // tokens of a sub-tile: its LDS parts grow with the waves
    constexpr int WB = SB < 8 ? SB : 8, SUBS = TT / WB;  // tokens of a walk, whose decays and states are in registers
    __shared__ __attribute__((aligned(16))) float s_d[3][TT][64];       // dt, dt u, gy
    __shared__ __attribute__((aligned(16))) float s_bc[TT][NW][8];
    __shared__ __attribute__((aligned(16))) float s_p[3][NW][SB][64];   // a wave's sums over its states: dh B, p A, C h

    const int nblk = a.G * a.blocks;
    const int64_t work = blockIdx.x / nblk;
    const int cb = (int)(blockIdx.x - work * nblk);
    SsmSeg sg;
    ssm_segment(a, work, sg);
    const int Dg = a.Dm / a.G, grp = cb / a.blocks, c0 = (cb - grp * a.blocks) * 64;
    const int lane = threadIdx.x & 63, w = wave_index(), n0 = NS * w;
    const bool chv = c0 + lane < Dg;
    const int ch = grp * Dg + (chv ? c0 + lane : 0);
    const int cl = (threadIdx.x % LPR) * V, tl = threadIdx.x / LPR;
    const bool lv = c0 + cl < Dg && (TS <= TT || tl < TT);
    const int lch = grp * Dg + (lv ? c0 + cl : 0);
    const int bn = threadIdx.x % (4 * NW), bt = threadIdx.x / (4 * NW);
    const T* pu = (const T*)a.u.p + sg.seq * a.u.sb + sg.t0 * a.u.st;
    const T* pd = (const T*)a.dl.p + sg.seq * a.dl.sb + sg.t0 * a.dl.st;
    const T* pz = a.z.p ? (const T*)a.z.p + sg.seq * a.z.sb + sg.t0 * a.z.st : nullptr;
    const T* py = (const T*)g.dy.p + sg.seq * g.dy.sb + sg.t0 * g.dy.st;
    const T* pB = (const T*)a.B + sg.seq * a.b_sb + sg.t0 * a.b_st + grp * a.b_sg;
    const T* pC = (const T*)a.C + sg.seq * a.c_sb + sg.t0 * a.c_st + grp * a.c_sg;
    const int64_t out0 = (sg.seq * a.T + sg.t0) * a.Dm;  // the segment's first row of du, ddelta, dz
    T *qu = (T*)g.du + out0, *qd = (T*)g.ddl + out0, *qz = pz ? (T*)g.dz + out0 : nullptr;

    float A[NS], Al[NS], e[NS], dA[NS], bias[V], Dv[V], dD[V], db[V];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        const bool ok = chv && n0 + j < a.N;  // lanes without a channel add zeros to dB and dC
        const float Aj = ok ? a.A[(int64_t)ch * a.N + n0 + j] : 0.f;
        A[j] = slope_decay(Aj);
        Al[j] = log2_decay(Aj);
        dA[j] = e[j] = 0.f;
        if (ok && a.nseg > 1) e[j] = a.ws_state[(work * a.N + n0 + j) * a.Dm + ch];
        else if (ok && g.dfin) e[j] = g.dfin[(sg.seq * a.Dm + ch) * a.N + n0 + j];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        bias[j] = a.bias ? a.bias[lch + j] : 0.f;
        Dv[j] = a.D ? a.D[lch + j] : 0.f;
        dD[j] = db[j] = 0.f;
    }
    Vec<T, V> ru[K], rd[K], rz[K], ry[K];
    Vec<T, 1> rb[KB], rc[KB];
    Vec<float, 1> rk[NS];
    const int vu = lv ? (tl * (int)a.u.st + lch) * ES : TILE_SKIP, vd = lv ? (tl * (int)a.dl.st + lch) * ES : TILE_SKIP;
    const int vz = lv ? (tl * (int)a.z.st + lch) * ES : TILE_SKIP, vy = lv ? (tl * (int)g.dy.st + lch) * ES : TILE_SKIP;
    const int vo = lv ? (tl * a.Dm + lch) * ES : TILE_SKIP;
    const int vb = bn < a.N ? (bt * (int)a.b_st + bn) * ES : TILE_SKIP;
    const int vc = bn < a.N ? (bt * (int)a.c_st + bn) * ES : TILE_SKIP;
    const int64_t nck = (a.T + TT - 1) / TT;
    auto fetch = [&](int t0) {
        const int left = t0 < 0 ? 0 : sg.len - t0;
        tile_load_rows(tile_rows(pu + t0 * a.u.st, a.u.st, left, a.Dm), vu, TS * ES * (int)a.u.st, ru);
        tile_load_rows(tile_rows(pd + t0 * a.dl.st, a.dl.st, left, a.Dm), vd, TS * ES * (int)a.dl.st, rd);
        tile_load_rows(tile_rows(py + t0 * g.dy.st, g.dy.st, left, a.Dm), vy, TS * ES * (int)g.dy.st, ry);
        tile_load_rows(tile_rows(pz ? pz + t0 * a.z.st : pz, a.z.st, left, a.Dm), vz, TS * ES * (int)a.z.st, rz);
        tile_load_rows(tile_rows(pB + t0 * a.b_st, a.b_st, left, a.N), vb, 16 * ES * (int)a.b_st, rb);
        tile_load_rows(tile_rows(pC + t0 * a.c_st, a.c_st, left, a.N), vc, 16 * ES * (int)a.c_st, rc);
        const auto kr = tile_rows(a.ckpt + (sg.seq * nck + (sg.t0 + t0) / TT) * a.N * a.Dm, a.Dm, left > 0 ? a.N : 0, a.Dm);
#pragma unroll
        for (int j = 0; j < NS; ++j) rk[j] = tile_load<float, 1>(kr, chv && n0 + j < a.N ? ((n0 + j) * a.Dm + ch) * 4 : TILE_SKIP);
    };
    const int live = (a.N + 3) >> 2;
    const int tiles = (sg.len + TT - 1) / TT;
    fetch((tiles - 1) * TT);
    {   // as in the forward: stores that write nothing, as many as a tile makes
        const float none[3 * K][V] = {};
        tile_store_rows<T>(tile_rows(qu, 0, 0, 0), TILE_SKIP, 0, none);
    }
    for (int k = tiles - 1; k >= 0; --k) {
        const int t0 = k * TT;
        Vec<T, V> cu[K], cd[K], cz[K], cy[K];
#pragma unroll
        for (int i = 0; i < K; ++i) {
            float dt[V], du[V], gy[V];
            cu[i] = ru[i], cd[i] = rd[i], cz[i] = rz[i], cy[i] = ry[i];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float x = (float)rd[i].v[j] + bias[j];
                dt[j] = a.softplus ? softplus(x) : x;
                gy[j] = (float)ry[i].v[j];
                if (pz) gy[j] *= silu_gate((float)rz[i].v[j]);
                du[j] = dt[j] * (float)ru[i].v[j];
            }
            if (t0 + i * TS + tl >= sg.len) {  // past the end: no step and no upstream
#pragma unroll
                for (int j = 0; j < V; ++j) dt[j] = du[j] = gy[j] = 0.f;
            }
            if (TS <= TT || tl < TT) {
                lds_store<V>(&s_d[0][i * TS + tl][cl], dt);
                lds_store<V>(&s_d[1][i * TS + tl][cl], du);
                lds_store<V>(&s_d[2][i * TS + tl][cl], gy);
            }
        }
#pragma unroll
        for (int i = 0; i < KB; ++i) {
            const bool in = t0 + i * 16 + bt < sg.len;
            s_bc[i * 16 + bt][bn >> 2][bn & 3] = in ? (float)rb[i].v[0] : 0.f;
            s_bc[i * 16 + bt][bn >> 2][4 + (bn & 3)] = in ? (float)rc[i].v[0] : 0.f;
        }
        float hs[SUBS][NS];  // the state that each walk starts from
#pragma unroll
        for (int j = 0; j < NS; ++j) hs[0][j] = rk[j].v[0];
        fetch(t0 - TT);
        __syncthreads();
        if (n0 < a.N) {
#pragma unroll
            for (int s = 0; s + 1 < SUBS; ++s) {
#pragma unroll
                for (int j = 0; j < NS; ++j) hs[s + 1][j] = hs[s][j];
#pragma unroll 1
                for (int t = s * WB; t < s * WB + WB; t += 4) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float dt = s_d[0][t + i][lane], du = s_d[1][t + i][lane];
                        const f32x4 b = *reinterpret_cast<const f32x4*>(&s_bc[t + i][w][0]);
#pragma unroll
                        for (int j = 0; j < NS; ++j)
                            hs[s + 1][j] = __builtin_fmaf(__builtin_amdgcn_exp2f(dt * Al[j]), hs[s + 1][j], du * b[j]);
                    }
                }
            }
        }
        // this tile's rows of part_bc
        const auto pr = tile_rows(g.part_bc + ((int64_t)cb * a.n_seqs * a.T + sg.seq * a.T + sg.t0 + t0) * (8 * NW), 8 * NW,
                                  sg.len - t0, 8 * NW);
#pragma unroll
        for (int s = SUBS - 1; s >= 0; --s) {
            if (n0 < a.N) {
                float av[WB][NS], hv[WB][NS];
#pragma unroll
                for (int t = 0; t < WB; ++t) {
                    const float dt = s_d[0][s * WB + t][lane], du = s_d[1][s * WB + t][lane];
                    const f32x4 b = *reinterpret_cast<const f32x4*>(&s_bc[s * WB + t][w][0]);
#pragma unroll
                    for (int j = 0; j < NS; ++j) {
                        av[t][j] = __builtin_amdgcn_exp2f(dt * Al[j]);
                        hv[t][j] = __builtin_fmaf(av[t][j], t ? hv[t - 1][j] : hs[s][j], du * b[j]);
                    }
                }
                reread();
                float keep = 0.f;
#pragma unroll
                for (int t = WB - 1; t >= 0; --t) {
                    const float dt = s_d[0][s * WB + t][lane], du = s_d[1][s * WB + t][lane], gy = s_d[2][s * WB + t][lane];
                    const f32x4 b = *reinterpret_cast<const f32x4*>(&s_bc[s * WB + t][w][0]);
                    const f32x4 c = *reinterpret_cast<const f32x4*>(&s_bc[s * WB + t][w][4]);
                    float v[8], s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
                    for (int j = 0; j < NS; ++j) {
                        const float dh = __builtin_fmaf(c[j], gy, e[j]);
                        v[j] = dh * du;
                        v[4 + j] = gy * hv[t][j];
                        s1 = j ? __builtin_fmaf(dh, b[j], s1) : dh * b[0];
                        s3 = j ? __builtin_fmaf(c[j], hv[t][j], s3) : c[0] * hv[t][0];
                        e[j] = dh * av[t][j];
                        const float p = e[j] * (t ? hv[t - 1][j] : hs[s][j]);
                        s2 = j ? __builtin_fmaf(p, A[j], s2) : p * A[0];
                        dA[j] = __builtin_fmaf(p, dt, dA[j]);
                    }
                    s_p[0][w][(s * WB + t) % SB][lane] = s1;
                    s_p[1][w][(s * WB + t) % SB][lane] = s2;
                    s_p[2][w][(s * WB + t) % SB][lane] = s3;
                    const float r = lanes_sum8(v);  // of value lane / 8, in all eight lanes
                    keep = t == WB - 1 || (lane & 7) == t ? r : keep;
                    if (t == 0) {
                        const float o[1] = {keep};
                        constexpr int ROW = 8 * NW * 4;
                        tile_store<float, 1>(o, pr, (lane & 7) < WB ? (s * WB + (lane & 7)) * ROW + (w * 8 + (lane >> 3)) * 4 : TILE_SKIP);
                    }
                    if ((t & 1) == 0) reread();
                }
            }
            if (s * WB % SB != 0) continue;  // a sub-tile's walks are done
            constexpr int WPS = SB / WB;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < K; ++i) {
                // threads past the tile's tokens have no sub-tile
                if (SB % TS == 0 ? i * TS / SB != s / WPS : (i * TS + tl) / SB != s / WPS) continue;
                const int t = i * TS + tl, ts = t % SB;
                float s1[V], s2[V], s3[V], o[V];
#pragma unroll
                for (int j = 0; j < V; ++j) s1[j] = s2[j] = s3[j] = 0.f;
                for (int q = 0; q < live; ++q) {
                    lds_add<V>(&s_p[0][q][ts][cl], s1);
                    lds_add<V>(&s_p[1][q][ts][cl], s2);
                    lds_add<V>(&s_p[2][q][ts][cl], s3);
                }
                float dt[V], gy[V];
#pragma unroll
                for (int j = 0; j < V; ++j) dt[j] = gy[j] = 0.f;
                lds_add<V>(&s_d[0][t][cl], dt);
                lds_add<V>(&s_d[2][t][cl], gy);
                const int at = vo + i * TS * a.Dm * ES;
                const int left = sg.len - t0;
                const int64_t r0 = (int64_t)t0 * a.Dm;
#pragma unroll
                for (int j = 0; j < V; ++j) o[j] = __builtin_fmaf(s1[j], dt[j], Dv[j] * gy[j]);
                tile_store<T, V>(o, tile_rows(qu + r0, a.Dm, left, a.Dm), at);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float uu = (float)cu[i].v[j];
                    o[j] = __builtin_fmaf(s1[j], uu, s2[j]);
                    if (a.softplus) o[j] *= fast_sigmoid((float)cd[i].v[j] + bias[j]);
                    dD[j] = __builtin_fmaf(gy[j], uu, dD[j]);
                    db[j] += t0 + t < sg.len ? o[j] : 0.f;
                }
                tile_store<T, V>(o, tile_rows(qd + r0, a.Dm, left, a.Dm), at);
                if (pz) {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float z = (float)cz[i].v[j], sz = fast_sigmoid(z);
                        o[j] = (float)cy[i].v[j] * __builtin_fmaf(Dv[j], (float)cu[i].v[j], s3[j]) * sz *
                               __builtin_fmaf(z, 1.f - sz, 1.f);
                    }
                }
                tile_store<T, V>(o, tile_rows(qz ? qz + r0 : qz, a.Dm, left, a.Dm), at);
            }
            __syncthreads();
        }
    }
    // the channel's dD and dbias: the classes of tokens that threads had, in order
    constexpr int ROWS = TS < TT ? TS : TT;
    if (TS <= TT || tl < TT) {
        lds_store<V>(&s_d[0][tl][cl], dD);
        lds_store<V>(&s_d[1][tl][cl], db);
    }
    __syncthreads();
    if (!chv) return;
    float* pp = g.part_par + work * (a.N + 2) * a.Dm + ch;
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        if (n0 + j >= a.N) continue;
        pp[(int64_t)(n0 + j) * a.Dm] = dA[j];
        if (a.nseg == 1 && g.ds0) g.ds0[(sg.seq * a.Dm + ch) * a.N + n0 + j] = e[j];
    }
    if (w == 0) {
        float s1 = 0.f, s2 = 0.f;
        for (int q = 0; q < ROWS; ++q) s1 += s_d[0][q][lane], s2 += s_d[1][q][lane];
        pp[(int64_t)a.N * a.Dm] = s1;
        pp[(int64_t)(a.N + 1) * a.Dm] = s2;
    }
}

// The parts added in a fixed order.  The first bc_blocks blocks: dB, dC over channel blocks, one thread per
// (token, group, state).  The others: dA, dD, dbias over work items, sixteen threads per (row, channel),
// each every sixteenth item, then these.
template <typename T>
__global__ __launch_bounds__(1024) void ssm_bwd_sum_kernel(SsmBwdParams g, int nw, int bc_blocks) {
    const SsmParams& a = g.f;
    __shared__ float red[16][64];
    if (blockIdx.x < bc_blocks) {
        const int64_t toks = a.n_seqs * a.T, id = (int64_t)blockIdx.x * 1024 + threadIdx.x;
        if (id >= toks * a.G * a.N) return;
        const int64_t tg = id / a.N, tok = tg / a.G;
        const int n = (int)(id - tg * a.N), grp = (int)(tg - tok * a.G);
        const float* p = g.part_bc + (((int64_t)grp * a.blocks * toks + tok) * nw + (n >> 2)) * 8 + (n & 3);
        float sb = 0.f, sc = 0.f;
#pragma unroll 4
        for (int k = 0; k < a.blocks; ++k) {
            sb += p[k * toks * nw * 8];
            sc += p[k * toks * nw * 8 + 4];
        }
        ((T*)g.dB)[id] = (T)sb;
        ((T*)g.dC)[id] = (T)sc;
        return;
    }
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t per = (int64_t)(a.N + 2) * a.Dm, id = (int64_t)(blockIdx.x - bc_blocks) * 64 + l;
    float s = id < per ? sum_parts(g.part_par + id, per, w, a.n_work) : 0.f;
    red[w][l] = s;
    __syncthreads();
    if (w || id >= per) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) s += red[i][l];
    const int n = (int)(id / a.Dm), ch = (int)(id - (int64_t)n * a.Dm);
    if (n < a.N) g.dA[(int64_t)ch * a.N + n] = s;
    else if (n == a.N) { if (g.dD) g.dD[ch] = s; }
    else if (g.dbias) g.dbias[ch] = s;
}

template <typename T, int V>
static hipError_t bwd_states_waves(const SsmBwdParams& g, hipStream_t s) {
    const dim3 grid((unsigned)(g.f.n_work * g.f.G * g.f.blocks));
    switch (ssm_waves(g.f.N)) {
        case 1: ssm_bwd_states_kernel<T, 1, V><<<grid, 64, 0, s>>>(g); break;
        case 2: ssm_bwd_states_kernel<T, 2, V><<<grid, 128, 0, s>>>(g); break;
        case 4: ssm_bwd_states_kernel<T, 4, V><<<grid, 256, 0, s>>>(g); break;
        case 8: ssm_bwd_states_kernel<T, 8, V><<<grid, 512, 0, s>>>(g); break;
        default: ssm_bwd_states_kernel<T, 16, V><<<grid, 1024, 0, s>>>(g); break;
    }
    return hipGetLastError();
}

template <typename T, int V>
static hipError_t bwd_waves(const SsmBwdParams& g, hipStream_t s) {
    const dim3 grid((unsigned)(g.f.n_work * g.f.G * g.f.blocks));
    switch (ssm_waves(g.f.N)) {
        case 1: ssm_bwd_kernel<T, 1, V><<<grid, 64, 0, s>>>(g); break;
        case 2: ssm_bwd_kernel<T, 2, V><<<grid, 128, 0, s>>>(g); break;
        case 4: ssm_bwd_kernel<T, 4, V><<<grid, 256, 0, s>>>(g); break;
        case 8: ssm_bwd_kernel<T, 8, V><<<grid, 512, 0, s>>>(g); break;
        default: ssm_bwd_kernel<T, 16, V><<<grid, 1024, 0, s>>>(g); break;
    }
    return hipGetLastError();
}

static bool by_four(const SsmBwdParams& g, int dt) {
    const SsmTok out{g.du, 0, 0}, out2{g.ddl, 0, 0}, out3{g.dz, 0, 0};
    return ssm_by_four(g.f.Dm / g.f.G, dt, {g.f.u, g.f.dl, g.f.z, g.dy, out, out2, out3});
}

hipError_t launch_ssm_bwd_states(const SsmBwdParams& g, int dt, hipStream_t s) {
    const bool v4 = by_four(g, dt);
    if (dt == DT_F32) return v4 ? bwd_states_waves<float, 4>(g, s) : bwd_states_waves<float, 1>(g, s);
    if (dt == DT_BF16) return v4 ? bwd_states_waves<__bf16, 4>(g, s) : bwd_states_waves<__bf16, 1>(g, s);
    return v4 ? bwd_states_waves<_Float16, 4>(g, s) : bwd_states_waves<_Float16, 1>(g, s);
}

hipError_t launch_ssm_bwd(const SsmBwdParams& g, int dt, hipStream_t s) {
    const bool v4 = by_four(g, dt);
    if (dt == DT_F32) return v4 ? bwd_waves<float, 4>(g, s) : bwd_waves<float, 1>(g, s);
    if (dt == DT_BF16) return v4 ? bwd_waves<__bf16, 4>(g, s) : bwd_waves<__bf16, 1>(g, s);
    return v4 ? bwd_waves<_Float16, 4>(g, s) : bwd_waves<_Float16, 1>(g, s);
}

hipError_t launch_ssm_bwd_sum(const SsmBwdParams& g, int dt, hipStream_t s) {
    const int64_t n = g.f.n_seqs * g.f.T * g.f.G * g.f.N, m = (int64_t)(g.f.N + 2) * g.f.Dm;
    const int nw = ssm_waves(g.f.N), bc = (int)((n + 1023) / 1024);
    const dim3 grid((unsigned)(bc + (m + 63) / 64));
    if (dt == DT_F32) ssm_bwd_sum_kernel<float><<<grid, 1024, 0, s>>>(g, nw, bc);
    else if (dt == DT_BF16) ssm_bwd_sum_kernel<__bf16><<<grid, 1024, 0, s>>>(g, nw, bc);
    else ssm_bwd_sum_kernel<_Float16><<<grid, 1024, 0, s>>>(g, nw, bc);
    return hipGetLastError();
}

}  // namespace triune
