// abi_ssm.hip -- extern "C" entry points of the state space layer's operators (declared in
// include/triune_hip.h): argument checks, workspace layout and launches.
#include "../../include/triune_hip.h"
#include "abi_common.h"
#include "ssm.h"

using namespace triune;

namespace {

// The kernels address a tile's 32 rows by 32-bit byte offsets.
constexpr int64_t kMaxTokenStride = 1 << 22;
bool strides_ok(std::initializer_list<int64_t> st) {
    for (const int64_t s : st)
        if (s < 0 || s >= kMaxTokenStride) return false;
    return true;
}

bool ssm_shape_ok(int64_t Dm, int64_t G, int N) {
    return Dm > 0 && Dm < kMaxTokenStride && G > 0 && Dm % G == 0 && N > 0 && N <= SSM_MAX_N;
}
// Workgroups that the channels of one group take, of all groups.
int64_t group_blocks(int64_t Dm, int64_t G) { return (Dm / G + 63) / 64; }
int64_t all_blocks(int64_t Dm, int64_t G) { return G * group_blocks(Dm, G); }

// The grids of a scan: its work items, and the join's.
bool scan_grids_ok(bool packed, int64_t n_work, int64_t nseg, int64_t n_seqs, int64_t Dm, int64_t G, int N) {
    if (!grid_ok(n_work, all_blocks(Dm, G), 64 * ssm_waves(N)) || n_seqs > kMaxGrid / (Dm * N)) return false;
    if (nseg <= 1) return true;
    const CarryGrid g = ssm_carry_grid(packed, n_seqs, n_work, nseg, Dm, N);
    return grid_ok(g.blocks, 1, 64 * g.waves);
}

// A chip's worth of workgroups is eight waves a compute unit (four SIMDs); two waves on a SIMD keep it three quarters
// busy.  Calls below the shares here split the time axis, which costs the decays a second time: unsplit they
// take as long for one workgroup as for the whole chip, split their time follows the work.  bf16, 8 x 2048 tokens, us
// unsplit and split, by workgroups:
//   outputs    N = 16: 256 230 234, 320 305 302, 352 304 320, 448 307 395, 504 308 446;  N = 8: 512 346 335,
//              640 348 427;  N = 32: 128 295 260, 160 296 333;  N = 64: 128 591 541, 160 591 725
//   gradients  N = 16: 320 1052 844, 400 1058 1006, 448 1058 1099, 504 1067 1240;  N = 8: 640 1522 1487, 768 1544 1761;
//              N = 32: 192 1231 1188, 240 1236 1457;  N = 64: 160 3549 2975, 240 3738 4337
// Split calls take shares that several rounds of workgroups even out: 1 x 16384 of 768 channels 106 us for
// 24 to 48 waves (segments of 128 and 64 tokens), 122 for 16; 16 ragged prompts of 5034 tokens, 1536 channels: 86 for
// 32, 91 for 24, 97 for 14, 87 for 64.
constexpr int kEnoughWaves = 8, kSplitWaves = 32;
constexpr int kForwardShare = 10, kGradientShare = 13;  // sixteenths of the chip's workgroups
// Workgroups of `waves` waves a compute unit.
int64_t ssm_slots(int N, int waves) {
    const int nw = ssm_waves(N);
    return (int64_t)compute_units() * (nw >= waves ? 1 : waves / nw);
}

int forced_segment(int flags) { return ((flags >> TRIUNE_FLAG_SEG_SHIFT) & 0xff) * SSM_UNIT; }

// Tokens of a segment of a dense call (a multiple of SSM_UNIT; the whole sequence unless splitting
// pays).  Two segments pay only where the sequence is short: `least` is the number that its length has to give, of
// which the chip has to hold three (gradients of 192 workgroups at N = 64: 4229 us in two segments, 3650 unsplit).
int64_t dense_segment(int64_t n_seqs, int64_t T, int64_t blocks, int N, int flags, int share, int64_t least) {
    const int64_t whole = (T + SSM_UNIT - 1) / SSM_UNIT * SSM_UNIT;
    if (forced_segment(flags)) return forced_segment(flags) < whole ? forced_segment(flags) : whole;
    if (16 * n_seqs * blocks >= share * ssm_slots(N, kEnoughWaves)) return whole;
    int64_t n = ssm_slots(N, kSplitWaves) / (n_seqs * blocks);
    if (n < 3) return whole;
    const int64_t most = T / 64;
    if (n > most) n = most;
    if (n < least) return whole;
    return ((T + n - 1) / n + SSM_UNIT - 1) / SSM_UNIT * SSM_UNIT;
}

struct ScanPlan {
    int64_t seg, nseg, n_work, cut;
    size_t off_sum, off_seg, total;
};

void plan_bytes(ScanPlan& p, int64_t Dm, int N, int64_t n_off) {
    p.off_sum = p.off_seg = p.total = 0;
    if (p.nseg <= 1) return;
    p.off_sum = align_up((size_t)p.n_work * N * Dm * 4);
    p.off_seg = p.off_sum + align_up((size_t)p.n_work * Dm * 4);
    p.total = p.off_seg + align_up((size_t)n_off * 4);
}

ScanPlan plan_scan(int64_t n_seqs, int64_t T, int64_t Dm, int64_t G, int N, int flags, bool gradients = false) {
    ScanPlan p{};
    p.seg = dense_segment(n_seqs, T, all_blocks(Dm, G), N, flags, gradients ? kGradientShare : kForwardShare,
                          gradients ? 2 : 3);
    p.nseg = (T + p.seg - 1) / p.seg;
    p.n_work = n_seqs * p.nseg;
    plan_bytes(p, Dm, N, 0);
    return p;
}

// Packed: lengths are on the device, so a segment is an equal share of all tokens.  Where there are sequences enough
// for two rounds of the chip they fill it by themselves, but for one far longer than the rest, which its
// workgroups would walk alone: sequences up to twice a workgroup's share of one round stay whole, and longer ones are
// cut into halves of it.  1536 channels, N = 16, bf16, us with every sequence whole and by this rule: 42 prompts of 64
// tokens and one of 16384 1730 and 259, and one of 2048 251 and 78; 200 of 100 and one of 8000 1047 and 341; 48
// log-uniform up to 8192 1139 and 965, 64 up to 2048 341 and 364.  Even lengths pay the launches that find
// nothing to do: 43 of 512 166 and 174, 200 of 256 308 and 312, 256 of 64 111 and 127, 64 of 100 57 and 66, so calls
// of few tokens stay whole (100 of 30: 37 and 45).  nseg > 1 says that there are segments.
ScanPlan plan_packed(int64_t n_seqs, int64_t total, int64_t Dm, int64_t G, int N, int flags) {
    ScanPlan p{};
    const int64_t blocks = all_blocks(Dm, G), slots = ssm_slots(N, kSplitWaves);
    p.seg = forced_segment(flags);
    if (!p.seg) {
        p.seg = (total * blocks / slots + SSM_UNIT - 1) / SSM_UNIT * SSM_UNIT;
        if (p.seg < 64) p.seg = 64;
        const int64_t round = ssm_slots(N, kEnoughWaves);
        if (n_seqs * blocks >= 2 * round) {
            const int64_t share = total * blocks / round < 256 ? 256 : total * blocks / round;
            p.seg = (share / 2 + SSM_UNIT - 1) / SSM_UNIT * SSM_UNIT;
            p.cut = total <= 4096 ? total : 2 * share;
        }
    }
    if (p.cut < p.seg) p.cut = p.seg;
    p.nseg = p.cut < total ? 2 : 1;
    p.n_work = p.nseg > 1 ? total / p.seg + n_seqs : n_seqs;
    plan_bytes(p, Dm, N, n_seqs + 1);
    return p;
}

struct BwdPlan {
    ScanPlan s;
    size_t off_bc, off_par, total;
};

BwdPlan plan_bwd(int64_t Bn, int64_t T, int64_t Dm, int64_t G, int N, int flags) {
    BwdPlan p{};
    p.s = plan_scan(Bn, T, Dm, G, N, flags, true);
    p.off_bc = p.s.total;
    p.off_par = p.off_bc + align_up((size_t)all_blocks(Dm, G) * Bn * T * ssm_waves(N) * 8 * 4);
    p.total = p.off_par + align_up((size_t)p.s.n_work * (N + 2) * Dm * 4);
    return p;
}

void set_sizes(SsmParams& a, int64_t n_seqs, int64_t T, int64_t Dm, int64_t G, int N, const ScanPlan& p, char* ws) {
    a.n_seqs = n_seqs;
    a.T = T;
    a.Dm = (int)Dm;
    a.G = (int)G;
    a.N = N;
    a.blocks = (int)group_blocks(Dm, G);
    a.seg = (int)p.seg;
    a.nseg = (int)p.nseg;
    a.n_work = p.n_work;
    if (p.nseg > 1) {
        a.ws_state = (float*)ws;
        a.ws_sum = (float*)(ws + p.off_sum);
    }
}

}  // namespace

extern "C" {

size_t triune_hip_ssm_scan_workspace_size(int64_t Bn, int64_t T, int64_t Dm, int64_t G, int N, int flags) {
    if (Bn <= 0 || T <= 0 || !tokens_ok(Bn, T) || !ssm_shape_ok(Dm, G, N)) return 0;
    return plan_scan(Bn, T, Dm, G, N, flags).total;
}

int triune_hip_ssm_scan(const void* u, const void* delta, const void* z, const void* B, const void* C, const float* A,
                        const float* D, const float* delta_bias, int io_dtype, const int64_t* strides, int softplus,
                        const float* s0, void* y, float* s_final, float* kept, int64_t Bn, int64_t T, int64_t Dm,
                        int64_t G, int N, int flags, void* workspace, size_t workspace_bytes, void* stream) {
    if (!u || !delta || !B || !C || !A || !y || !strides) return TRIUNE_ERR_NULL;
    if (!dtype_ok(io_dtype)) return TRIUNE_ERR_DTYPE;
    if (!tokens_ok(Bn, T) || !ssm_shape_ok(Dm, G, N)) return TRIUNE_ERR_SHAPE;
    if (!all_aligned(io_dtype, {u, delta, z, B, C, y}) ||
        !all_aligned(TRIUNE_DT_F32, {A, D, delta_bias, s0, s_final, kept}))
        return TRIUNE_ERR_LAYOUT;
    if (!strides_ok({strides[1], strides[3], strides[5], strides[7], strides[9], strides[12]}) || strides[7] < Dm)
        return TRIUNE_ERR_LAYOUT;
    if (Bn == 0) return TRIUNE_OK;
    if (T == 0) {
        if (!s_final) return TRIUNE_OK;
        return status(launch_state_copy(s0, s_final, Bn * Dm * N, 4, (hipStream_t)stream));
    }
    const ScanPlan p = plan_scan(Bn, T, Dm, G, N, flags);
    if (!scan_grids_ok(false, p.n_work, p.nseg, Bn, Dm, G, N)) return TRIUNE_ERR_SHAPE;
    if (const int e = check_ws(workspace, workspace_bytes, p.total)) return e;
    SsmParams a{};
    a.u = {u, strides[0], strides[1]};
    a.dl = {delta, strides[2], strides[3]};
    a.z = {z, strides[4], strides[5]};
    a.y = {y, strides[6], strides[7]};
    a.B = B, a.b_sb = strides[8], a.b_st = strides[9], a.b_sg = strides[10];
    a.C = C, a.c_sb = strides[11], a.c_st = strides[12], a.c_sg = strides[13];
    a.A = A, a.D = D, a.bias = delta_bias, a.softplus = softplus;
    a.s0 = s0, a.fin = s_final, a.ckpt = kept;
    set_sizes(a, Bn, T, Dm, G, N, p, (char*)workspace);
    const hipStream_t s = (hipStream_t)stream;
    if (p.nseg > 1) {
        if (const int e = status(launch_ssm_states(a, io_dtype, s))) return e;
        if (const int e = status(launch_ssm_carry(a, s))) return e;
    }
    return status(launch_ssm_scan(a, io_dtype, s));
}

size_t triune_hip_ssm_scan_varlen_workspace_size(int64_t n_seqs, int64_t total_tokens, int64_t Dm, int64_t G, int N,
                                                 int flags) {
    if (n_seqs <= 0 || total_tokens <= 0 || !tokens_ok(n_seqs, total_tokens) || !ssm_shape_ok(Dm, G, N)) return 0;
    return plan_packed(n_seqs, total_tokens, Dm, G, N, flags).total;
}

int triune_hip_ssm_scan_varlen(const void* u, const void* delta, const void* z, const void* B, const void* C,
                               const float* A, const float* D, const float* delta_bias, int io_dtype,
                               const int64_t* strides, int softplus, const int32_t* cu_seqlens, int64_t n_seqs,
                               int64_t total_tokens, const float* s0, float* s_final, const int32_t* slots,
                               int64_t n_state_rows, void* y, int64_t Dm, int64_t G, int N, int flags,
                               void* workspace, size_t workspace_bytes, void* stream) {
    if (!u || !delta || !B || !C || !A || !y || !strides || !cu_seqlens) return TRIUNE_ERR_NULL;
    if (!dtype_ok(io_dtype)) return TRIUNE_ERR_DTYPE;
    if (!tokens_ok(n_seqs, total_tokens) || n_state_rows < 0 || !ssm_shape_ok(Dm, G, N)) return TRIUNE_ERR_SHAPE;
    if (!slots && (s0 || s_final) && n_state_rows < n_seqs) return TRIUNE_ERR_SHAPE;
    if (!all_aligned(io_dtype, {u, delta, z, B, C, y}) ||
        !all_aligned(TRIUNE_DT_F32, {A, D, delta_bias, s0, s_final, cu_seqlens, slots}))
        return TRIUNE_ERR_LAYOUT;
    if (!strides_ok({strides[0], strides[1], strides[2], strides[3], strides[4], strides[6]}) || strides[3] < Dm)
        return TRIUNE_ERR_LAYOUT;
    if (n_seqs == 0) return TRIUNE_OK;
    // with no tokens every sequence's state still passes through: one empty segment each
    const ScanPlan p = plan_packed(n_seqs, total_tokens > 0 ? total_tokens : 1, Dm, G, N, flags);
    if (!scan_grids_ok(true, p.n_work, p.nseg, n_seqs, Dm, G, N)) return TRIUNE_ERR_SHAPE;
    if (const int e = check_ws(workspace, workspace_bytes, p.total)) return e;
    SsmParams a{};
    a.u = {u, 0, strides[0]};
    a.dl = {delta, 0, strides[1]};
    a.z = {z, 0, strides[2]};
    a.y = {y, 0, strides[3]};
    a.B = B, a.b_st = strides[4], a.b_sg = strides[5];
    a.C = C, a.c_st = strides[6], a.c_sg = strides[7];
    a.A = A, a.D = D, a.bias = delta_bias, a.softplus = softplus;
    a.s0 = s0, a.fin = s_final, a.slots = slots, a.n_slots = n_state_rows, a.cu = cu_seqlens;
    set_sizes(a, n_seqs, total_tokens, Dm, G, N, p, (char*)workspace);
    const hipStream_t s = (hipStream_t)stream;
    if (p.nseg > 1) {
        int32_t* off = (int32_t*)((char*)workspace + p.off_seg);
        if (const int e = status(launch_ssm_offsets(a, p.cut, off, s))) return e;
        a.seg_off = off;
        if (const int e = status(launch_ssm_states(a, io_dtype, s))) return e;
        if (const int e = status(launch_ssm_carry(a, s))) return e;
    }
    return status(launch_ssm_scan(a, io_dtype, s));
}

size_t triune_hip_ssm_bwd_workspace_size(int64_t Bn, int64_t T, int64_t Dm, int64_t G, int N, int flags) {
    if (Bn <= 0 || T <= 0 || !tokens_ok(Bn, T) || !ssm_shape_ok(Dm, G, N)) return 0;
    return plan_bwd(Bn, T, Dm, G, N, flags).total;
}

int triune_hip_ssm_bwd(const void* u, const void* delta, const void* z, const void* B, const void* C, const float* A,
                       const float* D, const float* delta_bias, const void* dy, int io_dtype, const int64_t* strides,
                       int softplus, const float* kept, const float* ds_final, void* du, void* ddelta, void* dz,
                       void* dB, void* dC, float* dA, float* dD, float* ddelta_bias, float* ds0, int64_t Bn, int64_t T,
                       int64_t Dm, int64_t G, int N, int flags, void* workspace, size_t workspace_bytes,
                       void* stream) {
    if (!u || !delta || !B || !C || !A || !dy || !strides || !kept || !du || !ddelta || (z && !dz) || !dB || !dC || !dA)
        return TRIUNE_ERR_NULL;
    if (!dtype_ok(io_dtype)) return TRIUNE_ERR_DTYPE;
    if (Bn <= 0 || T <= 0 || !tokens_ok(Bn, T) || !ssm_shape_ok(Dm, G, N)) return TRIUNE_ERR_SHAPE;
    if (!all_aligned(io_dtype, {u, delta, z, B, C, dy, du, ddelta, dz, dB, dC}) ||
        !all_aligned(TRIUNE_DT_F32, {A, D, delta_bias, kept, ds_final, dA, dD, ddelta_bias, ds0}))
        return TRIUNE_ERR_LAYOUT;
    if (!strides_ok({strides[1], strides[3], strides[5], strides[7], strides[9], strides[12]})) return TRIUNE_ERR_LAYOUT;
    const BwdPlan p = plan_bwd(Bn, T, Dm, G, N, flags);
    if (!scan_grids_ok(false, p.s.n_work, p.s.nseg, Bn, Dm, G, N) || Bn * T > kMaxGrid / (G * N)) return TRIUNE_ERR_SHAPE;
    if (const int e = check_ws(workspace, workspace_bytes, p.total)) return e;
    char* ws = (char*)workspace;
    SsmBwdParams g{};
    SsmParams& a = g.f;
    a.u = {u, strides[0], strides[1]};
    a.dl = {delta, strides[2], strides[3]};
    a.z = {z, strides[4], strides[5]};
    g.dy = {dy, strides[6], strides[7]};
    a.B = B, a.b_sb = strides[8], a.b_st = strides[9], a.b_sg = strides[10];
    a.C = C, a.c_sb = strides[11], a.c_st = strides[12], a.c_sg = strides[13];
    a.A = A, a.D = D, a.bias = delta_bias, a.softplus = softplus;
    a.ckpt = const_cast<float*>(kept);
    set_sizes(a, Bn, T, Dm, G, N, p.s, ws);
    g.dfin = ds_final;
    g.du = du, g.ddl = ddelta, g.dz = dz, g.dB = dB, g.dC = dC;
    g.part_bc = (float*)(ws + p.off_bc);
    g.part_par = (float*)(ws + p.off_par);
    g.dA = dA, g.dD = dD, g.dbias = ddelta_bias, g.ds0 = ds0;
    const hipStream_t s = (hipStream_t)stream;
    if (p.s.nseg > 1) {
        if (const int e = status(launch_ssm_bwd_states(g, io_dtype, s))) return e;
        if (const int e = status(launch_ssm_bwd_carry(g, s))) return e;
    }
    if (const int e = status(launch_ssm_bwd(g, io_dtype, s))) return e;
    return status(launch_ssm_bwd_sum(g, io_dtype, s));
}

int triune_hip_ssm_decode_step(const void* u, const void* delta, const void* z, const void* B, const void* C,
                               const float* A, const float* D, const float* delta_bias, int io_dtype,
                               const int64_t* strides, int softplus, const float* state_in, float* state_out,
                               const int32_t* slots, int64_t n_state_rows, void* y, int64_t Bn, int64_t Dm, int64_t G,
                               int N, void* stream) {
    if (!u || !delta || !B || !C || !A || !y || !strides || !state_in || !state_out) return TRIUNE_ERR_NULL;
    if (!dtype_ok(io_dtype)) return TRIUNE_ERR_DTYPE;
    if (Bn < 0 || n_state_rows < 0 || !ssm_shape_ok(Dm, G, N)) return TRIUNE_ERR_SHAPE;
    if (!slots && n_state_rows < Bn) return TRIUNE_ERR_SHAPE;
    if (!all_aligned(io_dtype, {u, delta, z, B, C, y}) ||
        !all_aligned(TRIUNE_DT_F32, {A, D, delta_bias, state_in, state_out, slots}))
        return TRIUNE_ERR_LAYOUT;
    if (Bn > kMaxGrid / ((Dm + 15) / 16)) return TRIUNE_ERR_SHAPE;
    if (Bn == 0) return TRIUNE_OK;
    SsmStepParams a{};
    a.u = {u, strides[0], 0};
    a.dl = {delta, strides[1], 0};
    a.z = {z, strides[2], 0};
    a.y = {y, strides[3], 0};
    a.B = B, a.b_sb = strides[4], a.b_sg = strides[5];
    a.C = C, a.c_sb = strides[6], a.c_sg = strides[7];
    a.A = A, a.D = D, a.bias = delta_bias, a.softplus = softplus;
    a.s_in = state_in, a.s_out = state_out, a.slots = slots, a.n_rows = n_state_rows;
    a.Bn = Bn, a.Dm = (int)Dm, a.G = (int)G, a.N = N, a.cus = compute_units();
    return status(launch_ssm_step(a, io_dtype, (hipStream_t)stream));
}

// ---- short convolution -------------------------------------------------------------------------
static int conv_check(const void* x, const void* w, const void* bias, const void* y, const int64_t* strides,
                      const void* s0, const void* fin, int io_dtype, int w_dtype, int64_t n, int64_t T, int64_t Dm,
                      int W) {
    if (!x || !w || !y || !strides) return TRIUNE_ERR_NULL;
    if (!dtype_ok(io_dtype) || (w_dtype != io_dtype && w_dtype != TRIUNE_DT_F32)) return TRIUNE_ERR_DTYPE;
    if (!tokens_ok(n, T) || Dm <= 0 || Dm >= (1 << 28) || W < 2 || W > 4) return TRIUNE_ERR_SHAPE;
    if (!all_aligned(io_dtype, {x, y, s0, fin}) || !all_aligned(w_dtype, {w, bias})) return TRIUNE_ERR_LAYOUT;
    // runs of 16 tokens x four channels, and (sequence, four channels) pairs, are numbered in 31 bits
    if (n > 0 && (Dm + 3) / 4 > kMaxGrid / (n * ((T + 15) / 16 + 1))) return TRIUNE_ERR_SHAPE;
    return TRIUNE_OK;
}

static ConvParams conv_params(const void* x, const void* w, const void* bias, int w_dtype, int silu, const void* s0,
                              void* fin, void* y, int64_t n, int64_t T, int64_t Dm, int W) {
    ConvParams a{};
    a.x = x, a.w = w, a.bias = bias, a.w_dt = w_dtype, a.silu = silu;
    a.s0 = s0, a.fin = fin, a.y = y, a.n_seqs = n, a.T = T, a.Dm = (int)Dm, a.W = W;
    return a;
}

int triune_hip_short_conv(const void* x, const void* w, const void* bias, int io_dtype, int w_dtype,
                          const int64_t* strides, int silu, const void* s0, void* s_final, void* y, int64_t Bn,
                          int64_t T, int64_t Dm, int W, void* stream) {
    if (const int e = conv_check(x, w, bias, y, strides, s0, s_final, io_dtype, w_dtype, Bn, T, Dm, W)) return e;
    if (Bn == 0) return TRIUNE_OK;
    if (T == 0) {
        if (!s_final) return TRIUNE_OK;
        const int bytes = io_dtype == TRIUNE_DT_F32 ? 4 : 2;
        return status(launch_state_copy(s0, s_final, Bn * (W - 1) * Dm, bytes, (hipStream_t)stream));
    }
    ConvParams a = conv_params(x, w, bias, w_dtype, silu, s0, s_final, y, Bn, T, Dm, W);
    a.x_sb = strides[0], a.x_st = strides[1], a.y_sb = strides[2], a.y_st = strides[3];
    a.run = conv_run(Bn, T, (int)Dm, compute_units());
    return status(launch_conv(a, io_dtype, (hipStream_t)stream));
}

int triune_hip_short_conv_varlen(const void* x, const void* w, const void* bias, int io_dtype, int w_dtype,
                                 const int64_t* strides, int silu, const int32_t* cu_seqlens, int64_t n_seqs,
                                 int64_t total_tokens, const void* s0, void* s_final, const int32_t* slots,
                                 int64_t n_state_rows, void* y, int64_t Dm, int W, void* stream) {
    if (const int e = conv_check(x, w, bias, y, strides, s0, s_final, io_dtype, w_dtype, n_seqs, total_tokens, Dm, W))
        return e;
    if (!cu_seqlens) return TRIUNE_ERR_NULL;
    if (n_state_rows < 0 || (!slots && (s0 || s_final) && n_state_rows < n_seqs)) return TRIUNE_ERR_SHAPE;
    if (!all_aligned(TRIUNE_DT_F32, {cu_seqlens, slots})) return TRIUNE_ERR_LAYOUT;
    if (n_seqs == 0) return TRIUNE_OK;
    ConvParams a = conv_params(x, w, bias, w_dtype, silu, s0, s_final, y, n_seqs, total_tokens, Dm, W);
    a.x_st = strides[0], a.y_st = strides[1];
    a.run = conv_run(1, total_tokens, (int)Dm, compute_units());
    a.cu = cu_seqlens, a.slots = slots, a.n_slots = n_state_rows;
    const hipStream_t s = (hipStream_t)stream;
    if (total_tokens > 0)
        if (const int e = status(launch_conv(a, io_dtype, s))) return e;
    return s_final ? status(launch_conv_state(a, io_dtype, s)) : TRIUNE_OK;
}

int triune_hip_short_conv_decode_step(const void* x, const void* w, const void* bias, int io_dtype, int w_dtype,
                                      const int64_t* strides, int silu, const void* state_in, void* state_out,
                                      const int32_t* slots, int64_t n_state_rows, void* y, int64_t Bn, int64_t Dm,
                                      int W, void* stream) {
    if (!state_in || !state_out) return TRIUNE_ERR_NULL;
    if (const int e = conv_check(x, w, bias, y, strides, state_in, state_out, io_dtype, w_dtype, Bn, 1, Dm, W))
        return e;
    if (n_state_rows < 0 || (!slots && n_state_rows < Bn)) return TRIUNE_ERR_SHAPE;
    if (!all_aligned(TRIUNE_DT_F32, {slots})) return TRIUNE_ERR_LAYOUT;
    if (Bn == 0) return TRIUNE_OK;
    ConvParams a = conv_params(x, w, bias, w_dtype, silu, state_in, state_out, y, Bn, 1, Dm, W);
    a.x_sb = strides[0], a.y_sb = strides[1];
    a.slots = slots, a.n_slots = n_state_rows;
    return status(launch_conv_step(a, io_dtype, (hipStream_t)stream));
}

size_t triune_hip_short_conv_bwd_workspace_size(int64_t Bn, int64_t T, int64_t Dm, int W) {
    if (Bn <= 0 || T <= 0 || !tokens_ok(Bn, T) || Dm <= 0 || Dm >= (1 << 28) || W < 2 || W > 4) return 0;
    const int run = conv_run(Bn, T, (int)Dm, compute_units());
    return align_up((size_t)conv_bwd_parts(Bn, T, (int)Dm, run) * (W + 1) * Dm * 4);
}

int triune_hip_short_conv_bwd(const void* x, const void* w, const void* bias, const void* dy, int io_dtype,
                              int w_dtype, const int64_t* strides, int silu, const void* s0, const void* ds_final,
                              void* dx, void* dw, void* dbias, void* ds0, int64_t Bn, int64_t T, int64_t Dm, int W,
                              void* workspace, size_t workspace_bytes, void* stream) {
    if (!dy) return TRIUNE_ERR_NULL;
    if (const int e = conv_check(x, w, bias, dx, strides, s0, ds0, io_dtype, w_dtype, Bn, T, Dm, W)) return e;
    if (!all_aligned(io_dtype, {dy, ds_final}) || !all_aligned(w_dtype, {dw, dbias})) return TRIUNE_ERR_LAYOUT;
    if (Bn == 0 || T == 0) return TRIUNE_ERR_SHAPE;
    ConvBwdParams g{};
    g.f = conv_params(x, w, bias, w_dtype, silu, s0, nullptr, nullptr, Bn, T, Dm, W);
    g.f.x_sb = strides[0], g.f.x_st = strides[1];
    g.dy = dy, g.dy_sb = strides[2], g.dy_st = strides[3];
    g.dfin = ds_final, g.dx = dx, g.ds0 = ds0;
    g.f.run = conv_run(Bn, T, (int)Dm, compute_units());
    g.parts = conv_bwd_parts(Bn, T, (int)Dm, g.f.run);
    if (dw || dbias) {
        if (const int e = check_ws(workspace, workspace_bytes, triune_hip_short_conv_bwd_workspace_size(Bn, T, Dm, W)))
            return e;
        g.part = (float*)workspace;
    }
    g.dw = dw, g.dbias = dbias;
    return status(launch_conv_bwd(g, io_dtype, (hipStream_t)stream));
}

// ---- layer norm ----------------------------------------------------------------------------------
static int norm_check(const void* x, const void* w, const void* b, int io_dtype, int w_dtype, int b_dtype, int64_t R,
                      int64_t D) {
    if (!x) return TRIUNE_ERR_NULL;
    if (!dtype_ok(io_dtype) || (w && w_dtype != io_dtype && w_dtype != TRIUNE_DT_F32) ||
        (b && b_dtype != io_dtype && b_dtype != TRIUNE_DT_F32))
        return TRIUNE_ERR_DTYPE;
    if (R < 0 || R > kMaxGrid || D <= 0 || D > NORM_MAX_D) return TRIUNE_ERR_SHAPE;
    if (!aligned(x, io_dtype) || !aligned(w, w_dtype) || !aligned(b, b_dtype)) return TRIUNE_ERR_LAYOUT;
    return TRIUNE_OK;
}

int triune_hip_layer_norm(const void* x, int64_t x_stride, const void* w, const void* b, int io_dtype, int w_dtype,
                          int b_dtype, float eps, void* y, float* mean, float* rstd, int64_t R, int64_t D,
                          void* stream) {
    if (!y || (mean == nullptr) != (rstd == nullptr)) return TRIUNE_ERR_NULL;
    if (const int e = norm_check(x, w, b, io_dtype, w_dtype, b_dtype, R, D)) return e;
    if (!aligned(y, io_dtype) || !all_aligned(TRIUNE_DT_F32, {mean, rstd})) return TRIUNE_ERR_LAYOUT;
    if (R == 0) return TRIUNE_OK;
    NormParams a{x, x_stride, w, b, w_dtype, b_dtype, eps, y, mean, rstd, R, (int)D, compute_units()};
    return status(launch_norm(a, io_dtype, (hipStream_t)stream));
}

size_t triune_hip_layer_norm_bwd_workspace_size(int64_t R, int64_t D) {
    if (R <= 0 || D <= 0 || D > NORM_MAX_D) return 0;
    return align_up((size_t)norm_bwd_parts(R, (int)D, compute_units()) * 2 * D * 4);
}

int triune_hip_layer_norm_bwd(const void* x, int64_t x_stride, const void* w, const void* dy, int64_t dy_stride,
                              int io_dtype, int w_dtype, int b_dtype, const float* mean, const float* rstd, void* dx,
                              void* dw, void* db, int64_t R, int64_t D, void* workspace, size_t workspace_bytes,
                              void* stream) {
    if (!dy || !mean || !rstd || !dx) return TRIUNE_ERR_NULL;
    if (const int e = norm_check(x, w, db, io_dtype, w_dtype, b_dtype, R, D)) return e;
    if (!all_aligned(io_dtype, {dy, dx}) || !all_aligned(TRIUNE_DT_F32, {mean, rstd}) || !aligned(dw, w_dtype))
        return TRIUNE_ERR_LAYOUT;
    if (R == 0) return TRIUNE_ERR_SHAPE;
    NormBwdParams g{};
    g.f = NormParams{x, x_stride, w, nullptr, w_dtype, b_dtype, 0.f, nullptr, const_cast<float*>(mean),
                     const_cast<float*>(rstd), R, (int)D, compute_units()};
    g.dy = dy, g.dy_st = dy_stride, g.dx = dx, g.dw = dw, g.db = db;
    g.parts = norm_bwd_parts(R, (int)D, compute_units());
    if (dw || db) {
        if (const int e = check_ws(workspace, workspace_bytes, (size_t)g.parts * 2 * D * 4)) return e;
        g.part = (float*)workspace;
    }
    return status(launch_norm_bwd(g, io_dtype, (hipStream_t)stream));
}

}  // extern "C"
