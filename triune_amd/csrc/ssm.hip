// ssm.hip -- the selective state space scan on gfx950: prompts, packed prompts and single tokens.
//
// For each channel d with states n:
//     dt_t = softplus(delta_t + bias);  h_t = exp(dt_t A_n) h_{t-1} + dt_t u_t B_t,n
//     y_t  = (sum_n C_t,n h_t,n + D u_t) silu(z_t)
// A channel's decays differ by state, so nothing of it factors into matrix products: each (token, channel,
// state) costs an exp2 and four plain operations, 23.5 cycles of a SIMD per wave measured (8.4 for the
// exp2; a plain operation 2.9 where two waves issue it, 5.5 alone, and 4.4 with a scalar or DPP
// operand), each (token, channel) about 200 more for softplus, gate, conversions and its LDS traffic.
// That, not the memory, bounds the kernel.
//
// Work split: a lane is a channel in the walk over the tokens, a wave holds four states of 64 channels
// in registers, a workgroup all states of 64 channels.  Tiles of tokens go through LDS: every (token,
// channel) is loaded and its softplus taken once for all states, by lanes of four channels, B and C are
// read as broadcasts, and the waves' parts of y meet there.  A form without that traffic (four lanes
// a channel, dt and dt u as DPP operands, y summed by DPP) issued as many operations, each slower:
// 437 us for 8 x 2048 tokens of 4096 channels (N = 16, bf16) against 306.
//
// Calls with too few (sequence, channel block) pairs for the chip split the time axis into segments: a
// pass for each segment's own end state but the last one's (its decay over the segment is exp(A sum dt), so only
// the sum of dt is kept), a scan over segments, and the pass that writes the outputs.
#include "ssm.h"

namespace triune {

// Waves of a workgroup, by the number of states: four states each.
int ssm_waves(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

// NW: waves; V: channels that a lane loads and stores together (4 where alignment allows); STATES: only
// the segment's end state from zero, and its sum of dt.
template <typename T, int NW, int V, bool STATES>
__global__ __launch_bounds__(64 * NW) void ssm_scan_kernel(SsmParams a) {
    constexpr int NS = 4, NT = 64 * NW;
    constexpr int TT = NW == 1 || NW == 16 ? 16 : 32;  // tokens of a tile: sixteen waves' parts of y fill the LDS
    constexpr int LPR = 64 / V;                        // lanes of a token's row
    constexpr int TS = NT / LPR;                       // tokens of one access of the workgroup
    constexpr int K = (TT + TS - 1) / TS;              // accesses of a tile
    constexpr int KB = TT * 4 * NW / NT;               // elements of B (and C) that a thread loads
    constexpr int BW = STATES ? NS : 2 * NS;
    constexpr int U = 2;                               // tokens whose operands are read together
    constexpr int ES = sizeof(T);
    __shared__ __attribute__((aligned(16))) float s_d[2][TT][64];       // dt, dt u
    __shared__ __attribute__((aligned(16))) float s_bc[TT][NW][BW];     // a wave's B, then its C
    __shared__ __attribute__((aligned(16))) float s_y[STATES ? 1 : NW][STATES ? 1 : TT][64];

    const int nblk = a.G * a.blocks;
    int64_t work = blockIdx.x / nblk;
    const int cb = (int)(blockIdx.x - work * nblk);
    int64_t seq = -1;
    if (STATES && a.cu) {
        seq = ssm_followed(a, work);
        if (seq < 0) return;
        work += seq;
    }
    SsmSeg sg;
    if (!ssm_segment(a, work, sg, seq)) return;
    if (STATES && sg.last) return;  // nothing follows that would start from its end
    const int Dg = a.Dm / a.G, grp = cb / a.blocks, c0 = (cb - grp * a.blocks) * 64;
    const int lane = threadIdx.x & 63, w = wave_index(), n0 = NS * w;
    // the walk's channel; lanes past the group's channels repeat its first and store nothing
    const bool chv = c0 + lane < Dg;
    const int ch = grp * Dg + (chv ? c0 + lane : 0);
    // the channels and the first token that this thread loads and stores, of a tile
    const int cl = (threadIdx.x % LPR) * V, tl = threadIdx.x / LPR;
    const bool lv = c0 + cl < Dg && (TS <= TT || tl < TT);
    const int lch = grp * Dg + (lv ? c0 + cl : 0);
    // the state and the first token that it loads B and C of
    const int bn = threadIdx.x % (4 * NW), bt = threadIdx.x / (4 * NW);

    const int64_t tok = sg.row0 + sg.t0, bat = a.cu ? 0 : sg.seq;
    const T* pu = (const T*)a.u.p + bat * a.u.sb + tok * a.u.st;
    const T* pd = (const T*)a.dl.p + bat * a.dl.sb + tok * a.dl.st;
    const T* pz = a.z.p ? (const T*)a.z.p + bat * a.z.sb + tok * a.z.st : nullptr;
    T* py = (T*)const_cast<void*>(a.y.p) + bat * a.y.sb + tok * a.y.st;
    const T* pB = (const T*)a.B + bat * a.b_sb + tok * a.b_st + grp * a.b_sg;
    const T* pC = (const T*)a.C + bat * a.c_sb + tok * a.c_st + grp * a.c_sg;

    float Al[NS], h[NS], bias[V], Dv[V];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        Al[j] = n0 + j < a.N ? log2_decay(a.A[(int64_t)ch * a.N + n0 + j]) : 0.f;
        h[j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        bias[j] = a.bias ? a.bias[lch + j] : 0.f;
        Dv[j] = a.D ? a.D[lch + j] : 0.f;
    }
    const int64_t row = STATES ? 0 : ssm_row(a.slots, a.n_slots, sg.seq);
    if constexpr (!STATES) {
        if (a.ws_state && !(sg.last && sg.index == 0)) {  // of several: its entering state comes from the join
#pragma unroll
            for (int j = 0; j < NS; ++j)
                if (n0 + j < a.N) h[j] = a.ws_state[(work * a.N + n0 + j) * a.Dm + ch];
        } else if (a.s0 && row >= 0) {
#pragma unroll
            for (int j = 0; j < NS; ++j)
                if (n0 + j < a.N) h[j] = a.s0[(row * a.Dm + ch) * a.N + n0 + j];
        }
        if (n0 >= a.N)  // waves without states add nothing to y
            for (int t = 0; t < TT; ++t) s_y[w][t][lane] = 0.f;
    }

    // A tile's loads, issued a tile ahead.
    Vec<T, V> ru[K], rd[K], rz[STATES ? 1 : K];
    Vec<T, 1> rb[KB], rc[STATES ? 1 : KB];
    const int vu = lv ? (tl * (int)a.u.st + lch) * ES : TILE_SKIP, vd = lv ? (tl * (int)a.dl.st + lch) * ES : TILE_SKIP;
    const int vz = lv ? (tl * (int)a.z.st + lch) * ES : TILE_SKIP, vy = lv ? (tl * (int)a.y.st + lch) * ES : TILE_SKIP;
    const int vb = bn < a.N ? (bt * (int)a.b_st + bn) * ES : TILE_SKIP;
    const int vc = bn < a.N ? (bt * (int)a.c_st + bn) * ES : TILE_SKIP;
    auto fetch = [&](int t0) {
        const int left = sg.len - t0;
        tile_load_rows(tile_rows(pu + t0 * a.u.st, a.u.st, left, a.Dm), vu, TS * ES * (int)a.u.st, ru);
        tile_load_rows(tile_rows(pd + t0 * a.dl.st, a.dl.st, left, a.Dm), vd, TS * ES * (int)a.dl.st, rd);
        tile_load_rows(tile_rows(pB + t0 * a.b_st, a.b_st, left, a.N), vb, 16 * ES * (int)a.b_st, rb);
        if constexpr (!STATES) {
            tile_load_rows(tile_rows(pz ? pz + t0 * a.z.st : pz, a.z.st, left, a.Dm), vz, TS * ES * (int)a.z.st, rz);
            tile_load_rows(tile_rows(pC + t0 * a.c_st, a.c_st, left, a.N), vc, 16 * ES * (int)a.c_st, rc);
        }
    };
    struct Block {
        float dt[U], du[U], b[U][BW];
    };
    auto read = [&](Block& x, int t) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            x.dt[i] = s_d[0][t + i][lane];
            x.du[i] = s_d[1][t + i][lane];
#pragma unroll
            for (int j = 0; j < BW; ++j) x.b[i][j] = s_bc[t + i][w][j];
        }
    };
    auto walk = [&](const Block& x, int t) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            float y = 0.f;
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                h[j] = __builtin_fmaf(__builtin_amdgcn_exp2f(x.dt[i] * Al[j]), h[j], x.du[i] * x.b[i][j]);
                if constexpr (!STATES) y = j ? __builtin_fmaf(x.b[i][NS + j], h[j], y) : x.b[i][NS] * h[0];
            }
            if constexpr (!STATES) s_y[w][t + i][lane] = y;
        }
    };
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.f;
    fetch(0);
    if constexpr (!STATES) {
        // Stores that write nothing, so that the loop is entered with as many accesses after its first
        // loads as it has on its way round: else those loads would be waited for together with a
        // tile's stores, which come after them.
        const float none[K][V] = {};
        tile_store_rows<T>(tile_rows(py, 0, 0, 0), TILE_SKIP, 0, none);
    }
    for (int t0 = 0; t0 < sg.len; t0 += TT) {
        const bool whole = t0 + TT <= sg.len;
        Vec<T, V> cu[STATES ? 1 : K], cz[STATES ? 1 : K];
        float dt[K][V], du[K][V];
#pragma unroll
        for (int i = 0; i < K; ++i) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                dt[i][j] = (float)rd[i].v[j] + bias[j];
                du[i][j] = (float)ru[i].v[j];
            }
            if constexpr (!STATES) cu[i] = ru[i], cz[i] = rz[i];
        }
        if (a.softplus) {
#pragma unroll
            for (int i = 0; i < K; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) dt[i][j] = softplus(dt[i][j]);
        }
#pragma unroll
        for (int i = 0; i < K; ++i) {
#pragma unroll
            for (int j = 0; j < V; ++j) du[i][j] *= dt[i][j];
            if (!whole && t0 + i * TS + tl >= sg.len) {  // past the end: no step, which leaves the state as it is
#pragma unroll
                for (int j = 0; j < V; ++j) dt[i][j] = du[i][j] = 0.f;
            }
            if (TS <= TT || tl < TT) {
                lds_store<V>(&s_d[0][i * TS + tl][cl], dt[i]);
                lds_store<V>(&s_d[1][i * TS + tl][cl], du[i]);
            }
            if constexpr (STATES) {
#pragma unroll
                for (int j = 0; j < V; ++j) sum[j] += TS <= TT || tl < TT ? dt[i][j] : 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < KB; ++i) {
            const bool in = whole || t0 + i * 16 + bt < sg.len;
            s_bc[i * 16 + bt][bn >> 2][bn & 3] = in ? (float)rb[i].v[0] : 0.f;
            if constexpr (!STATES) s_bc[i * 16 + bt][bn >> 2][NS + (bn & 3)] = (float)rc[i].v[0];
        }
        fetch(t0 + TT);
        constexpr int EVERY = NW == 16 ? 16 : 32;  // ssm_kept_every
        if (!STATES && a.ckpt && chv && (sg.t0 + t0) % EVERY == 0) {
            const int64_t nck = (a.T + EVERY - 1) / EVERY, ck = sg.seq * nck + (sg.t0 + t0) / EVERY;
#pragma unroll
            for (int j = 0; j < NS; ++j)
                if (n0 + j < a.N) a.ckpt[(ck * a.N + n0 + j) * a.Dm + ch] = h[j];
        }
        __syncthreads();
        if (n0 < a.N) {
            Block p, q;  // read one block ahead
            read(p, 0);
#pragma unroll 1
            for (int t = 0; t < TT; t += 2 * U) {
                read(q, t + U);
                walk(p, t);
                read(p, t + 2 * U < TT ? t + 2 * U : 0);
                walk(q, t + U);
            }
        }
        __syncthreads();
        if constexpr (!STATES) {
            float y[K][V];
#pragma unroll
            for (int i = 0; i < K; ++i) {
#pragma unroll
                for (int j = 0; j < V; ++j) y[i][j] = Dv[j] * (float)cu[i].v[j];
                if (TS > TT && tl >= TT) continue;
#pragma unroll
                for (int k = 0; k < NW; ++k) lds_add<V>(&s_y[k][i * TS + tl][cl], y[i]);
            }
            if (pz) {
#pragma unroll
                for (int i = 0; i < K; ++i)
#pragma unroll
                    for (int j = 0; j < V; ++j) y[i][j] *= silu_gate((float)cz[i].v[j]);
            }
            tile_store_rows<T>(tile_rows(py + t0 * a.y.st, a.y.st, sg.len - t0, a.Dm), vy, TS * ES * (int)a.y.st, y);
        }
    }
    if constexpr (STATES) {
        if (chv) {
#pragma unroll
            for (int j = 0; j < NS; ++j)
                if (n0 + j < a.N) a.ws_state[(work * a.N + n0 + j) * a.Dm + ch] = h[j];
        }
        constexpr int ROWS = TS < TT ? TS : TT;
        if (TS <= TT || tl < TT) lds_store<V>(&s_d[0][tl][cl], sum);  // every wave is past its reads of s_d
        __syncthreads();
        if (w == 0 && chv) {
            float s = 0.f;
            for (int k = 0; k < ROWS; ++k) s += s_d[0][k][lane];
            a.ws_sum[work * a.Dm + ch] = s;
        }
    } else if (a.fin && sg.last && row >= 0 && chv) {
#pragma unroll
        for (int j = 0; j < NS; ++j)
            if (n0 + j < a.N) a.fin[(row * a.Dm + ch) * a.N + n0 + j] = h[j];
    }
}

// The scan over a sequence's segments: each one's own end state is replaced by the state that it starts
// from (BACK: from the last to the first, each one's own gradient at its start by the one that enters at
// its end).  A block takes 64 channels of a (sequence, state), its waves eight segments each at a time:
// a wave folds its segments to one, the folds meet in LDS, and each wave finishes from the state that the
// waves before it leave.  128 segments of 768 channels, N = 16: 7.6 us, 6.9 with decays that may overflow (Pow2);
// a thread per channel with eight segments in flight 15.7.
template <bool BACK>
__global__ __launch_bounds__(1024) void ssm_carry_kernel(SsmParams a, const float* init, float* out, bool by_followed) {
    constexpr int PER = 8;  // segments of a wave
    __shared__ float s_m[16][64], s_end[16][64];  // a wave's decay (mantissa, exponent) and its end from zero
    __shared__ int s_e[16][64];
    const int lane = threadIdx.x & 63, w = wave_index(), waves = blockDim.x >> 6;
    const int cb = (a.Dm + 63) / 64;
    const int64_t sn = blockIdx.x / cb;
    int64_t seq = sn / a.N;
    const int n = (int)(sn - seq * a.N), c = (int)(blockIdx.x - sn * cb) * 64 + lane;
    if (by_followed) {  // the block of a sequence's first segment takes the sequence
        const int64_t j = seq;
        seq = ssm_followed(a, j);
        if (seq < 0 || a.seg_off[seq] - seq != j) return;
    }
    const bool chv = c < a.Dm;
    const int ch = chv ? c : 0;
    const int64_t per = (int64_t)a.N * a.Dm, at = (int64_t)ch * a.N + n;
    int64_t first = seq * a.nseg, count = a.nseg;
    if (a.cu) first = a.seg_off[seq], count = min((int64_t)a.seg_off[seq + 1], a.n_work) - first;
    if (a.cu && count == 1) return;
    const int64_t from = BACK ? count : count - 1;  // segments whose own result is there
    const float Al = log2_decay(a.A[at]);
    const int64_t row = ssm_row(a.slots, a.n_slots, seq);
    float S = init && row >= 0 ? init[row * per + at] : 0.f;
    float* p = a.ws_state + (int64_t)n * a.Dm + ch;
    const float* ps = a.ws_sum + ch;
    for (int64_t k0 = 0; k0 < count; k0 += PER * waves) {
        float local[PER], sum[PER];
        const int64_t k = k0 + PER * w;
        const int m = (int)max(min(count - k, (int64_t)PER), (int64_t)0);  // segments that this wave has
        const int64_t v0 = BACK ? first + count - 1 - k : first + k;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int64_t v = BACK ? v0 - i : v0 + i;
            local[i] = k + i < from ? p[v * per] : 0.f;
            sum[i] = k + i < from ? ps[v * a.Dm] : 0.f;
        }
        float all = 0.f, end = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            end = Pow2(sum[i] * Al).scale(end) + local[i];
            all += sum[i];
        }
        const Pow2 own(all * Al);
        if (waves > 1) {
            s_m[w][lane] = own.m;
            s_e[w][lane] = own.e;
            s_end[w][lane] = end;
            __syncthreads();
        }
        float next = S;
        for (int q = 0; q < waves; ++q) {
            if (q == w) S = next;
            next = waves > 1 ? Pow2(s_m[q][lane], s_e[q][lane]).scale(next) + s_end[q][lane] : own.scale(next) + end;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (i < m && chv) p[(BACK ? v0 - i : v0 + i) * per] = S;
            S = Pow2(sum[i] * Al).scale(S) + local[i];
        }
        S = next;
        if (waves > 1) __syncthreads();
    }
    if (out && w == 0 && chv) out[row * per + at] = S;
}

// Packed calls: seg_off[i] = segments of the sequences before i (one at least for each).  One wave.
__global__ __launch_bounds__(64) void ssm_offsets_kernel(SsmParams a, int64_t cut, int32_t* off) {
    const int lane = threadIdx.x;
    int64_t base = 0;
    if (lane == 0) off[0] = 0;
    for (int64_t i0 = 0; i0 < a.n_seqs; i0 += 64) {
        const int64_t i = i0 + lane;
        int64_t n = 0;
        if (i < a.n_seqs) {
            const int64_t beg = min(max((int64_t)a.cu[i], (int64_t)0), a.T);
            const int64_t len = min(max((int64_t)a.cu[i + 1], beg), a.T) - beg;
            n = len > cut ? (len + a.seg - 1) / a.seg : 1;
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

template <typename T>
__global__ __launch_bounds__(256) void state_copy_kernel(const T* from, T* to, int64_t n) {
    const int64_t step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += step) to[i] = from ? from[i] : (T)0;
}

// One token for every row.  A lane holds up to four states of a channel, LPC neighbouring lanes a
// channel; a block keeps its channels' A, D and bias over the rows that it walks, the next row's
// states and operands in flight.  Bound by the states, read and written once.
template <typename T, int LPC>
__global__ __launch_bounds__(256) void ssm_step_kernel(SsmStepParams a, int blocks) {
    constexpr int CPB = 256 / LPC;  // channels of a block
    const int ch = (int)(blockIdx.x % blocks) * CPB + threadIdx.x / LPC, q = threadIdx.x % LPC, n0 = 4 * q;
    const bool chv = ch < a.Dm;
    const int c = chv ? ch : 0, left = chv ? a.N - n0 : 0, grp = c / (a.Dm / a.G);
    float Al[4];
    load_states<4>(a.A + (int64_t)c * a.N + n0, left, Al);
#pragma unroll
    for (int j = 0; j < 4; ++j) Al[j] = log2_decay(Al[j]);
    const float bias = a.bias ? a.bias[c] : 0.f, Dv = a.D ? a.D[c] : 0.f;
    struct Row {
        int64_t row;
        float h[4];
        Raw<T, 4> B, C;
        T u, dl, z;
    } x;
    auto fetch = [&](int64_t b) {
        x.row = ssm_row(a.slots, a.n_rows, b);
        load_states<4>(a.s_in + (x.row * a.Dm + c) * a.N + n0, x.row >= 0 ? left : 0, x.h);
        x.B = load_raw<4>((const T*)a.B + b * a.b_sb + grp * a.b_sg + n0, left);
        x.C = load_raw<4>((const T*)a.C + b * a.c_sb + grp * a.c_sg + n0, left);
        x.u = ((const T*)a.u.p)[b * a.u.sb + c];
        x.dl = ((const T*)a.dl.p)[b * a.dl.sb + c];
        x.z = a.z.p ? ((const T*)a.z.p)[b * a.z.sb + c] : (T)0.f;
    };
    const int64_t step = gridDim.x / blocks;
    int64_t b = blockIdx.x / blocks;
    fetch(b);
    for (; b < a.Bn; b += step) {
        const Row r = x;
        if (b + step < a.Bn) fetch(b + step);
        const float uu = (float)r.u, xx = (float)r.dl + bias;
        const float dt = a.softplus ? softplus(xx) : xx, dtu = dt * uu;
        float h[4], y = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            h[j] = __builtin_fmaf(__builtin_amdgcn_exp2f(dt * Al[j]), r.h[j], dtu * (float)r.B.v[j]);
            y = __builtin_fmaf((float)r.C.v[j], h[j], y);
        }
        if (r.row >= 0 && left > 0) store_states<4>(a.s_out + (r.row * a.Dm + c) * a.N + n0, left, h);
        if constexpr (LPC >= 2) y = dpp_add<0xB1>(y);
        if constexpr (LPC >= 4) y = dpp_add<0x4E>(y);
        if constexpr (LPC >= 8) y = dpp_add<0x141>(y);
        if constexpr (LPC >= 16) y = dpp_add<0x140>(y);
        if (q == 0 && chv) {
            y = __builtin_fmaf(Dv, uu, y);
            if (a.z.p) y *= silu_gate((float)r.z);
            ((T*)const_cast<void*>(a.y.p))[b * a.y.sb + c] = (T)(r.row >= 0 ? y : 0.f);
        }
    }
}

template <typename T, int V, bool STATES>
static hipError_t scan_waves(const SsmParams& a, hipStream_t s) {
    const int64_t work = STATES && a.cu ? a.n_work - a.n_seqs : a.n_work;  // packed: those that another segment follows
    const dim3 grid((unsigned)(work * a.G * a.blocks));
    switch (ssm_waves(a.N)) {
        case 1: ssm_scan_kernel<T, 1, V, STATES><<<grid, 64, 0, s>>>(a); break;
        case 2: ssm_scan_kernel<T, 2, V, STATES><<<grid, 128, 0, s>>>(a); break;
        case 4: ssm_scan_kernel<T, 4, V, STATES><<<grid, 256, 0, s>>>(a); break;
        case 8: ssm_scan_kernel<T, 8, V, STATES><<<grid, 512, 0, s>>>(a); break;
        default: ssm_scan_kernel<T, 16, V, STATES><<<grid, 1024, 0, s>>>(a); break;
    }
    return hipGetLastError();
}

template <bool STATES>
static hipError_t scan_dtype(const SsmParams& a, int dt, hipStream_t s) {
    const bool v4 = ssm_by_four(a.Dm / a.G, dt, {a.u, a.dl, a.z, a.y});
    if (dt == DT_F32) return v4 ? scan_waves<float, 4, STATES>(a, s) : scan_waves<float, 1, STATES>(a, s);
    if (dt == DT_BF16) return v4 ? scan_waves<__bf16, 4, STATES>(a, s) : scan_waves<__bf16, 1, STATES>(a, s);
    return v4 ? scan_waves<_Float16, 4, STATES>(a, s) : scan_waves<_Float16, 1, STATES>(a, s);
}

hipError_t launch_ssm_states(const SsmParams& a, int dt, hipStream_t s) { return scan_dtype<true>(a, dt, s); }
hipError_t launch_ssm_scan(const SsmParams& a, int dt, hipStream_t s) { return scan_dtype<false>(a, dt, s); }

CarryGrid ssm_carry_grid(bool packed, int64_t n_seqs, int64_t n_work, int64_t nseg, int64_t Dm, int N) {
    // Waves for the segments of a sequence.  Packed calls know the average alone and take two waves from five segments
    // on: 16 ragged prompts of 5034 tokens (6 segments, the longest 23) 84 us a call with one wave, 81 with two,
    // 82 with four, 90 with eight; 20 of 300 tokens (6) 54, 56, 59, 68; three, one of them of 5000 (28), 62, 54,
    // 52, 51.
    const int64_t segs = packed ? (n_work + n_seqs - 1) / n_seqs : nseg;
    CarryGrid g;
    g.waves = segs <= (packed ? 4 : 8) ? 1 : segs <= 16 ? 2 : segs <= 32 ? 4 : segs <= 64 ? 8 : 16;
    // Packed: sequences of one segment need no join, so where fewer segments are followed by another than there are
    // sequences, blocks are laid out by those (256 prompts of 64 tokens: 127 us a call, 155 by sequences).
    g.by_followed = packed && n_work - n_seqs < n_seqs;
    g.blocks = (g.by_followed ? n_work - n_seqs : n_seqs) * N * ((Dm + 63) / 64);
    return g;
}

template <bool BACK>
static hipError_t carry(const SsmParams& a, const float* init, float* out, hipStream_t s) {
    const CarryGrid g = ssm_carry_grid(a.cu, a.n_seqs, a.n_work, a.nseg, a.Dm, a.N);
    ssm_carry_kernel<BACK><<<dim3((unsigned)g.blocks), 64 * g.waves, 0, s>>>(a, init, out, g.by_followed);
    return hipGetLastError();
}
hipError_t launch_ssm_carry(const SsmParams& a, hipStream_t s) { return carry<false>(a, a.s0, nullptr, s); }
hipError_t launch_ssm_bwd_carry(const SsmBwdParams& g, hipStream_t s) { return carry<true>(g.f, g.dfin, g.ds0, s); }

hipError_t launch_ssm_offsets(const SsmParams& a, int64_t cut, int32_t* off, hipStream_t s) {
    ssm_offsets_kernel<<<1, 64, 0, s>>>(a, cut, off);
    return hipGetLastError();
}

hipError_t launch_state_copy(const void* from, void* to, int64_t n, int bytes, hipStream_t s) {
    if (from == to || n == 0) return hipSuccess;
    const int64_t blocks = (n + 255) / 256;
    const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096));
    if (bytes == 4) state_copy_kernel<uint32_t><<<grid, 256, 0, s>>>((const uint32_t*)from, (uint32_t*)to, n);
    else state_copy_kernel<uint16_t><<<grid, 256, 0, s>>>((const uint16_t*)from, (uint16_t*)to, n);
    return hipGetLastError();
}

template <typename T>
static hipError_t step_lanes(const SsmStepParams& a, hipStream_t s) {
    const int lpc = a.N <= 4 ? 1 : a.N <= 8 ? 2 : a.N <= 16 ? 4 : a.N <= 32 ? 8 : 16;
    const int64_t blocks = (a.Dm * (int64_t)lpc + 255) / 256;
    // rows that are walked side by side: eight blocks a compute unit (256 sessions of 1536 channels, N = 16:
    // 14.9 us; 16.8 with four, 16.6 with sixteen, 19.1 with a block per row and 64 channels).  None of these divides
    // the rows evenly: 85 side by side leave the last of four rounds one row.  Even divisions have not been tried.
    int64_t rows = a.cus * 8 / blocks;
    rows = rows < 1 ? 1 : rows > a.Bn ? a.Bn : rows;
    const dim3 grid((unsigned)(blocks * rows));
    switch (lpc) {
        case 1: ssm_step_kernel<T, 1><<<grid, 256, 0, s>>>(a, (int)blocks); break;
        case 2: ssm_step_kernel<T, 2><<<grid, 256, 0, s>>>(a, (int)blocks); break;
        case 4: ssm_step_kernel<T, 4><<<grid, 256, 0, s>>>(a, (int)blocks); break;
        case 8: ssm_step_kernel<T, 8><<<grid, 256, 0, s>>>(a, (int)blocks); break;
        default: ssm_step_kernel<T, 16><<<grid, 256, 0, s>>>(a, (int)blocks); break;
    }
    return hipGetLastError();
}

hipError_t launch_ssm_step(const SsmStepParams& a, int dt, hipStream_t s) {
    if (dt == DT_F32) return step_lanes<float>(a, s);
    if (dt == DT_BF16) return step_lanes<__bf16>(a, s);
    return step_lanes<_Float16>(a, s);
}

}  // namespace triune
