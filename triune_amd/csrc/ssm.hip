// ssm.hip -- the selective state space scan on gfx950: prompts, packed prompts and single tokens.
//
// For each channel d with states n:
//     dt_t = softplus(delta_t + bias);  h_t = exp(dt_t A_n) h_{t-1} + dt_t u_t B_t,n
//     y_t  = (sum_n C_t,n h_t,n + D u_t) silu(z_t)
// A channel's decays differ by state, so nothing of it factors into matrix products: each (token,
// channel, state) costs an exp2 (8.5 cycles per wave on a SIMD, measured) and four plain
// operations, and that, not the memory, bounds the kernel.
//
// Work split: a lane is a channel, a wave holds four states of 64 channels in registers, a
// workgroup all states of 64 channels.  Tiles of 32 tokens go through LDS: every (token, channel)
// is loaded and its softplus taken once for all states (by one of the waves), B and C are read
// as broadcasts, and the waves' parts of y meet there.  Calls with too few (sequence, channel block) pairs
// for the chip split the time axis into segments: a pass for each segment's own end state (its
// decay over the segment is exp(A sum dt), so only the sum of dt is kept), a scan over segments, and
// the pass that writes the outputs.
#include "ssm.h"

namespace triune {

int ssm_waves(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

// STATES: only the segment's end state from zero, and its sum of dt.
template <typename T, int NW, bool STATES>
__global__ __launch_bounds__(64 * NW) void ssm_scan_kernel(SsmParams a) {
    constexpr int TT = NW == 16 ? 16 : 32;  // sixteen waves' parts of y for 32 tokens would fill the LDS
    constexpr int TPW = TT / NW;            // tokens a wave loads and stores
    constexpr int BW = STATES ? 4 : 8;
    __shared__ float2 s_du[TT][64];     // dt, dt u
    __shared__ float s_bc[TT][NW][BW];  // a wave's four B, then its four C
    __shared__ float s_y[STATES ? 1 : NW][STATES ? 1 : TT][64];

    const int nblk = a.G * a.blocks;
    const int64_t work = blockIdx.x / nblk;
    const int cb = (int)(blockIdx.x - work * nblk);
    SsmSeg sg;
    if (!ssm_segment(a, work, sg)) return;
    const int Dg = a.Dm / a.G, grp = cb / a.blocks;
    const int lane = threadIdx.x & 63, w = wave_index();
    const int in_grp = (cb - grp * a.blocks) * SSM_BLOCK + lane;
    const bool chv = in_grp < Dg;
    const int ch = grp * Dg + in_grp;
    const int n0 = 4 * w;

    const int64_t tok = sg.row0 + sg.t0, bat = a.cu ? 0 : sg.seq;
    const T* pu = (const T*)a.u.p + bat * a.u.sb + tok * a.u.st + (chv ? ch : 0);
    const T* pd = (const T*)a.dl.p + bat * a.dl.sb + tok * a.dl.st + (chv ? ch : 0);
    const T* pz = a.z.p ? (const T*)a.z.p + bat * a.z.sb + tok * a.z.st + (chv ? ch : 0) : nullptr;
    T* py = (T*)const_cast<void*>(a.y.p) + bat * a.y.sb + tok * a.y.st + (chv ? ch : 0);
    const T* pB = (const T*)a.B + bat * a.b_sb + tok * a.b_st + grp * a.b_sg;
    const T* pC = (const T*)a.C + bat * a.c_sb + tok * a.c_st + grp * a.c_sg;

    float Al[4], h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        Al[j] = chv && n0 + j < a.N ? a.A[(int64_t)ch * a.N + n0 + j] * LOG2E : 0.f;
        h[j] = 0.f;
    }
    const float bias = a.bias && chv ? a.bias[ch] : 0.f, Dv = a.D && chv ? a.D[ch] : 0.f;
    const int64_t row = STATES ? 0 : ssm_row(a.slots, a.n_slots, sg.seq);
    if (!STATES && chv) {
        if (a.ws_state) {  // segmented: the entering state comes from the scan over segments
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n0 + j < a.N) h[j] = a.ws_state[(work * a.N + n0 + j) * a.Dm + ch];
        } else if (a.s0 && row >= 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n0 + j < a.N) h[j] = a.s0[(row * a.Dm + ch) * a.N + n0 + j];
        }
    }

    T ru[TPW], rd[TPW], rz[STATES ? 1 : TPW];
    auto fetch = [&](int t0) {
#pragma unroll
        for (int i = 0; i < TPW; ++i) {
            const int t = t0 + i * NW + w;
            const bool ok = t < sg.len && chv;
            ru[i] = ok ? pu[t * a.u.st] : (T)0.f;
            rd[i] = ok ? pd[t * a.dl.st] : (T)0.f;
            if constexpr (!STATES) rz[i] = ok && pz ? pz[t * a.z.st] : (T)0.f;
        }
    };
    float sum = 0.f;
    fetch(0);
    for (int t0 = 0; t0 < sg.len; t0 += TT) {
        float cu[STATES ? 1 : TPW], cz[STATES ? 1 : TPW];
#pragma unroll
        for (int i = 0; i < TPW; ++i) {
            const int t = i * NW + w;
            const float x = (float)rd[i] + bias, uu = (float)ru[i];
            const float dt = t0 + t < sg.len ? (a.softplus ? softplus(x) : x) : 0.f;
            s_du[t][lane] = make_float2(dt, dt * uu);
            if constexpr (STATES) {
                sum += dt;
            } else {
                cu[i] = uu;
                cz[i] = (float)rz[i];
            }
        }
        for (int e = threadIdx.x; e < TT * 4 * NW; e += 64 * NW) {
            const int t = e / (4 * NW), n = e % (4 * NW);
            const bool ok = t0 + t < sg.len && n < a.N;
            s_bc[t][n >> 2][n & 3] = ok ? (float)pB[(t0 + t) * a.b_st + n] : 0.f;
            if constexpr (!STATES) s_bc[t][n >> 2][4 + (n & 3)] = ok ? (float)pC[(t0 + t) * a.c_st + n] : 0.f;
        }
        if (t0 + TT < sg.len) fetch(t0 + TT);
        if (!STATES && a.ckpt && chv && (sg.t0 + t0) % SSM_CKPT == 0) {
            const int64_t nck = (a.T + SSM_CKPT - 1) / SSM_CKPT, ck = sg.seq * nck + (sg.t0 + t0) / SSM_CKPT;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n0 + j < a.N) a.ckpt[(ck * a.N + n0 + j) * a.Dm + ch] = h[j];
        }
        __syncthreads();
        const int nt = min(TT, sg.len - t0);
        if (n0 < a.N) {
#pragma unroll 4
            for (int t = 0; t < nt; ++t) {
                const float2 d = s_du[t][lane];
                const f32x4 b = *reinterpret_cast<const f32x4*>(&s_bc[t][w][0]);
                float y = 0.f;
                f32x4 c;
                if constexpr (!STATES) c = *reinterpret_cast<const f32x4*>(&s_bc[t][w][4]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    h[j] = __builtin_fmaf(__builtin_amdgcn_exp2f(d.x * Al[j]), h[j], d.y * b[j]);
                    if constexpr (!STATES) y = __builtin_fmaf(c[j], h[j], y);
                }
                if constexpr (!STATES) s_y[w][t][lane] = y;
            }
        }
        __syncthreads();
        if constexpr (!STATES) {
            const int live = (a.N + 3) >> 2;  // waves that hold states
#pragma unroll
            for (int i = 0; i < TPW; ++i) {
                const int t = i * NW + w;
                float y = Dv * cu[i];
                for (int k = 0; k < live; ++k) y += s_y[k][t][lane];
                if (pz) y *= silu_gate(cz[i]);
                if (t0 + t < sg.len && chv) py[(t0 + t) * a.y.st] = (T)y;
            }
        }
    }
    if constexpr (STATES) {
        if (chv) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n0 + j < a.N) a.ws_state[(work * a.N + n0 + j) * a.Dm + ch] = h[j];
        }
        float* red = reinterpret_cast<float*>(&s_du[0][0]);  // every wave is past its reads of s_du
        red[w * 64 + lane] = sum;
        __syncthreads();
        if (w == 0 && chv) {
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < NW; ++k) s += red[k * 64 + lane];
            a.ws_sum[work * a.Dm + ch] = s;
        }
    } else if (a.fin && sg.last && row >= 0 && chv) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n0 + j < a.N) a.fin[(row * a.Dm + ch) * a.N + n0 + j] = h[j];
    }
}

// The scan over a sequence's segments: each one's own end state is replaced by the state it starts
// from.  One thread per (sequence, state, channel).
__global__ __launch_bounds__(256) void ssm_carry_kernel(SsmParams a) {
    const int64_t per = (int64_t)a.N * a.Dm, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= a.n_seqs * per) return;
    const int64_t seq = id / per;
    const int n = (int)((id - seq * per) / a.Dm), ch = (int)((id - seq * per) % a.Dm);
    int64_t w0 = seq * a.nseg, w1 = w0 + a.nseg;
    if (a.cu) w0 = a.seg_off[seq], w1 = min((int64_t)a.seg_off[seq + 1], a.n_work);
    const float Al = a.A[(int64_t)ch * a.N + n] * LOG2E;
    const int64_t row = ssm_row(a.slots, a.n_slots, seq);
    float S = a.s0 && row >= 0 ? a.s0[(row * a.Dm + ch) * a.N + n] : 0.f;
    for (int64_t w = w0; w < w1; ++w) {
        float* p = a.ws_state + w * per + (int64_t)n * a.Dm + ch;
        const float local = *p;
        *p = S;
        S = __builtin_fmaf(__builtin_amdgcn_exp2f(a.ws_sum[w * a.Dm + ch] * Al), S, local);
    }
}

// Packed calls: seg_off[i] = segments of the sequences before i (one at least for each).  One wave.
__global__ __launch_bounds__(64) void ssm_offsets_kernel(SsmParams a, int32_t* off) {
    const int lane = threadIdx.x;
    int64_t base = 0;
    if (lane == 0) off[0] = 0;
    for (int64_t i0 = 0; i0 < a.n_seqs; i0 += 64) {
        const int64_t i = i0 + lane;
        int64_t n = 0;
        if (i < a.n_seqs) {
            const int64_t beg = min(max((int64_t)a.cu[i], (int64_t)0), a.T);
            const int64_t len = min(max((int64_t)a.cu[i + 1], beg), a.T) - beg;
            n = max((len + a.seg - 1) / a.seg, (int64_t)1);
        }
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) {
            const int64_t o = __shfl_up(n, k);
            if (lane >= k) n += o;
        }
        if (i < a.n_seqs) off[i + 1] = (int32_t)min(base + n, a.n_work);
        base += __shfl(n, 63);
    }
}

// One token for every row.  A lane holds up to four states of a channel, LPC lanes a channel.
template <typename T, int LPC, bool VEC>
__global__ __launch_bounds__(256) void ssm_step_kernel(SsmStepParams a) {
    constexpr int CPB = 256 / LPC;  // channels of a block
    const int64_t nblk = (a.Dm + CPB - 1) / CPB;
    const int64_t b = blockIdx.x / nblk;
    const int ch = (int)(blockIdx.x - b * nblk) * CPB + threadIdx.x / LPC, q = threadIdx.x % LPC, n0 = 4 * q;
    const bool chv = ch < a.Dm;
    const int c = chv ? ch : 0;
    const int64_t row = ssm_row(a.slots, a.n_rows, b);
    float h[4] = {0.f, 0.f, 0.f, 0.f}, Al[4] = {0.f, 0.f, 0.f, 0.f};
    const bool live = chv && row >= 0 && n0 < a.N;
    if (live) {
        const float *ps = a.s_in + (row * a.Dm + c) * a.N + n0, *pA = a.A + (int64_t)c * a.N + n0;
        if constexpr (VEC) {
            const f32x4 s = *reinterpret_cast<const f32x4*>(ps), m = *reinterpret_cast<const f32x4*>(pA);
#pragma unroll
            for (int j = 0; j < 4; ++j) h[j] = s[j], Al[j] = m[j] * LOG2E;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n0 + j < a.N) h[j] = ps[j], Al[j] = pA[j] * LOG2E;
        }
    }
    const int grp = c / (a.Dm / a.G);
    const T *pB = (const T*)a.B + b * a.b_sb + grp * a.b_sg + n0, *pC = (const T*)a.C + b * a.c_sb + grp * a.c_sg + n0;
    const float x = (float)((const T*)a.dl.p)[b * a.dl.sb + c] + (a.bias ? a.bias[c] : 0.f);
    const float uu = (float)((const T*)a.u.p)[b * a.u.sb + c];
    const float dt = a.softplus ? softplus(x) : x, dtu = dt * uu;
    float y = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool ok = n0 + j < a.N;
        const float bb = ok ? (float)pB[j] : 0.f, cc = ok ? (float)pC[j] : 0.f;
        h[j] = __builtin_fmaf(__builtin_amdgcn_exp2f(dt * Al[j]), h[j], dtu * bb);
        y = __builtin_fmaf(cc, h[j], y);
    }
    if (live) {
        float* ps = a.s_out + (row * a.Dm + c) * a.N + n0;
        if constexpr (VEC) {
            *reinterpret_cast<f32x4*>(ps) = f32x4{h[0], h[1], h[2], h[3]};
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n0 + j < a.N) ps[j] = h[j];
        }
    }
    if constexpr (LPC >= 2) y = dpp_add<0xB1>(y);
    if constexpr (LPC >= 4) y = dpp_add<0x4E>(y);
    if constexpr (LPC >= 8) y = dpp_add<0x141>(y);
    if constexpr (LPC >= 16) y = dpp_add<0x140>(y);
    if (q == 0 && chv) {
        if (a.D) y = __builtin_fmaf(a.D[c], uu, y);
        if (a.z.p) y *= silu_gate((float)((const T*)a.z.p)[b * a.z.sb + c]);
        ((T*)const_cast<void*>(a.y.p))[b * a.y.sb + c] = (T)(row >= 0 ? y : 0.f);
    }
}

template <typename T, bool STATES>
static hipError_t scan_waves(const SsmParams& a, hipStream_t s) {
    const dim3 grid((unsigned)(a.n_work * a.G * a.blocks));
    switch (ssm_waves(a.N)) {
        case 1: ssm_scan_kernel<T, 1, STATES><<<grid, 64, 0, s>>>(a); break;
        case 2: ssm_scan_kernel<T, 2, STATES><<<grid, 128, 0, s>>>(a); break;
        case 4: ssm_scan_kernel<T, 4, STATES><<<grid, 256, 0, s>>>(a); break;
        case 8: ssm_scan_kernel<T, 8, STATES><<<grid, 512, 0, s>>>(a); break;
        default: ssm_scan_kernel<T, 16, STATES><<<grid, 1024, 0, s>>>(a); break;
    }
    return hipGetLastError();
}

template <bool STATES>
static hipError_t scan_dtype(const SsmParams& a, int dt, hipStream_t s) {
    if (dt == DT_F32) return scan_waves<float, STATES>(a, s);
    if (dt == DT_BF16) return scan_waves<__bf16, STATES>(a, s);
    return scan_waves<_Float16, STATES>(a, s);
}

hipError_t launch_ssm_states(const SsmParams& a, int dt, hipStream_t s) { return scan_dtype<true>(a, dt, s); }
hipError_t launch_ssm_scan(const SsmParams& a, int dt, hipStream_t s) { return scan_dtype<false>(a, dt, s); }

hipError_t launch_ssm_carry(const SsmParams& a, hipStream_t s) {
    const int64_t n = a.n_seqs * a.N * a.Dm;
    ssm_carry_kernel<<<dim3((unsigned)((n + 255) / 256)), 256, 0, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_ssm_offsets(const SsmParams& a, int32_t* off, hipStream_t s) {
    ssm_offsets_kernel<<<1, 64, 0, s>>>(a, off);
    return hipGetLastError();
}

template <typename T, bool VEC>
static hipError_t step_lanes(const SsmStepParams& a, hipStream_t s) {
    const int lpc = ssm_waves(a.N), cpb = 256 / lpc;
    const dim3 grid((unsigned)(a.Bn * ((a.Dm + cpb - 1) / cpb)));
    switch (lpc) {
        case 1: ssm_step_kernel<T, 1, VEC><<<grid, 256, 0, s>>>(a); break;
        case 2: ssm_step_kernel<T, 2, VEC><<<grid, 256, 0, s>>>(a); break;
        case 4: ssm_step_kernel<T, 4, VEC><<<grid, 256, 0, s>>>(a); break;
        case 8: ssm_step_kernel<T, 8, VEC><<<grid, 256, 0, s>>>(a); break;
        default: ssm_step_kernel<T, 16, VEC><<<grid, 256, 0, s>>>(a); break;
    }
    return hipGetLastError();
}

hipError_t launch_ssm_step(const SsmStepParams& a, int dt, hipStream_t s) {
    const bool vec = a.N % 4 == 0 && !((reinterpret_cast<uintptr_t>(a.s_in) | reinterpret_cast<uintptr_t>(a.s_out) |
                                        reinterpret_cast<uintptr_t>(a.A)) & 15);
    if (dt == DT_F32) return vec ? step_lanes<float, true>(a, s) : step_lanes<float, false>(a, s);
    if (dt == DT_BF16) return vec ? step_lanes<__bf16, true>(a, s) : step_lanes<__bf16, false>(a, s);
    return vec ? step_lanes<_Float16, true>(a, s) : step_lanes<_Float16, false>(a, s);
}

}  // namespace triune
