// abi_decay.hip -- extern "C" entry points of the decay attention layer's operators (declared in
// include/triune_hip.h): argument checks, workspace layout and launches.
#include "abi_common.h"
#include "decay.h"
#include "rms_norm.h"

using namespace triune;

namespace {

bool decay_shape_ok(int64_t H, int64_t Hk, int64_t Dk, int64_t Dv) {
    return H > 0 && H < (1 << 16) && Hk > 0 && H % Hk == 0 && Dk > 0 && Dk <= DECAY_MAX_DK && Dv > 0 &&
           Dv <= DECAY_MAX_DV;
}
int64_t slices_of(int64_t Dv) { return (Dv + decay_slice((int)Dv) - 1) / decay_slice((int)Dv); }

// Sequences whose workgroups are a grid: what the plans below multiply then stays within 64 bits.
bool seqs_ok(int64_t n_seqs, int64_t H, int64_t Dv) { return grid_ok(n_seqs, H * slices_of(Dv), 256); }

int forced_segment(int flags) { return ((flags >> TRIUNE_FLAG_SEG_SHIFT) & 0xff) * DECAY_CHUNK; }
int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

// Workgroups that split calls are cut into: three to every two compute units where a workgroup holds a whole state of more
// than 8192 values, three to each otherwise.  A cut costs a state written, joined and read, 16 bytes a value, a long
// segment leaves compute units idle.  Forward in us, bf16, by tokens a segment ([x]: what this takes):
//   4 x 16384, 6 heads of 64:     256 97.2, 384 95.7, [512] 85.4, 768 103.1
//   1 x 8192, 24 heads, 128 x 64: 128 84.9, [256] 68.8, 384 66.9, 512 75.9
//   4 x 2048, 12 heads of 128:    128 82.5, 192 78.8, [256] 72.1, 384 84.0
//   1 x 2048, 16 heads of 128:    64 48.1, [128] 39.8, 192 40.8, 256 47.6
//   2 x 512, 8 heads of 128:      [64] 26.4, 128 30.8, 256 42.1
// It loses most at 1 x 4096, 12 heads of 128 ([128] 54.7, 192 48.0) and 1 x 16384 of them ([512] 123.5, 768 118.2).
int64_t chip_slots(int64_t Dk, int64_t Dv) {
    return (int64_t)compute_units() * (decay_padded_dk((int)Dk) * decay_slice((int)Dv) > 8192 ? 3 : 6) / 2;
}
// The least tokens of a packed call's segment; its sequences end in shorter ones as they are.  Dense: 64, whole chunks of
// the gradients.
int64_t least_segment(int64_t Dk, int64_t Dv) {
    const int values = decay_padded_dk((int)Dk) * decay_slice((int)Dv);
    return values > 8192 ? 192 : values > 4096 ? 128 : 64;
}

struct DecayPlan {
    int64_t seg, nseg, n_work, cut;
    size_t off_sum, off_seg, total;
};

void plan_bytes(DecayPlan& p, int64_t H, int64_t Dk, int64_t Dv, int64_t n_off) {
    p.off_sum = p.off_seg = p.total = 0;
    if (p.nseg <= 1) return;
    p.off_sum = align_up((size_t)(p.n_work * H) * decay_state_values((int)Dk, (int)Dv) * 4);
    p.off_seg = p.off_sum + align_up((size_t)(p.n_work * H) * 8);
    p.total = p.off_seg + align_up((size_t)n_off * 4);
}

DecayPlan plan_dense(int64_t n_seqs, int64_t T, int64_t H, int64_t Dk, int64_t Dv, int flags) {
    DecayPlan p{};
    const int64_t whole = round_up(T, DECAY_CHUNK), blocks = n_seqs * H * slices_of(Dv);
    p.seg = forced_segment(flags);
    if (!p.seg) {
        int64_t n = chip_slots(Dk, Dv) / blocks;
        if (n > T / 64) n = T / 64;
        p.seg = n < 2 ? whole : (T + n - 1) / n;
    }
    p.seg = round_up(p.seg, 64);  // whole chunks of the gradients
    if (p.seg > whole) p.seg = whole;
    p.nseg = (T + p.seg - 1) / p.seg;
    p.n_work = n_seqs * p.nseg;
    plan_bytes(p, H, Dk, Dv, 0);
    return p;
}

// The grids of a call: its work items, and where there are segments the join's, four values of a state a thread.  States
// themselves are addressed in 64 bits.
bool grids_ok(const DecayPlan& p, int64_t n_seqs, int64_t H, int64_t Dk, int64_t Dv) {
    const int64_t values = decay_state_values((int)Dk, (int)Dv);
    return grid_ok(p.n_work, H * slices_of(Dv), 256) &&
           (p.nseg <= 1 || grid_ok(n_seqs, H * ((values + 1023) / 1024), 256));
}

// Packed: lengths are on the device, so a segment is an equal share of all tokens.  nseg > 1 says that there may be
// segments; sequences whose join would outgrow a grid are enough without them.
DecayPlan plan_packed(int64_t n_seqs, int64_t total, int64_t H, int64_t Dk, int64_t Dv, int flags) {
    DecayPlan p{};
    p.seg = forced_segment(flags);
    if (!p.seg) {
        p.seg = round_up(total * H * slices_of(Dv) / chip_slots(Dk, Dv), DECAY_CHUNK);
        if (p.seg < least_segment(Dk, Dv)) p.seg = least_segment(Dk, Dv);
        p.cut = p.seg * 3 / 2;
    }
    if (p.cut < p.seg) p.cut = p.seg;
    p.nseg = p.cut < total ? 2 : 1;
    p.n_work = p.nseg > 1 ? total / p.seg + n_seqs : n_seqs;
    if (!forced_segment(flags) && !grids_ok(p, n_seqs, H, Dk, Dv)) {
        p.nseg = 1;
        p.n_work = n_seqs;
    }
    plan_bytes(p, H, Dk, Dv, n_seqs + 1);
    return p;
}

// Gradients: the segments' end states of the states' gradients, the states of every chunk, sums of shared heads and of
// constant gates, and last the forward's end states, which take no place where the forward's workspace holds them.
struct GradPlan {
    DecayPlan p;
    int64_t chunk, nc;
    size_t off_S, off_R, off_q, off_k, off_g, off_ends, total;
};

GradPlan plan_grad(int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv, int io_dtype, int g_head,
                   int flags) {
    GradPlan r{};
    r.p = plan_dense(B, T, H, Dk, Dv, flags);
    r.chunk = decay_grad_chunk(io_dtype == TRIUNE_DT_BF16);
    r.nc = (T + r.chunk - 1) / r.chunk;
    const size_t heads = (size_t)(B * H), states = align_up(heads * r.nc * decay_state_values((int)Dk, (int)Dv) * 4);
    const size_t shared = H > Hk ? align_up((size_t)(B * T * H) * Dk * 4) : 0;
    r.off_S = r.p.total;
    r.off_R = r.off_S + states;
    r.off_q = r.off_R + states;
    r.off_k = r.off_q + shared;
    r.off_g = r.off_k + shared;
    r.off_ends = r.off_g + (g_head ? align_up(heads * r.nc * 4) : 0);
    r.total = r.off_ends + r.p.total;
    return r;
}

bool grad_grids_ok(const GradPlan& r, int64_t B, int64_t H, int64_t Dk, int64_t Dv) {
    return grids_ok(r.p, B, H, Dk, Dv) && grid_ok(B * r.nc, H, 256);
}

void set_sizes(DecayParams& a, int64_t n_seqs, int64_t T, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv,
               const DecayPlan& p, char* ws) {
    a.n_seqs = n_seqs;
    a.T = T;
    a.H = (int)H;
    a.per = (int)(H / Hk);
    a.Dk = (int)Dk;
    a.Dv = (int)Dv;
    a.slices = (int)slices_of(Dv);
    a.seg = (int)p.seg;
    a.nseg = (int)p.nseg;
    a.n_work = p.n_work;
    if (p.nseg > 1) {
        a.ws_state = (float*)ws;
        a.ws_sum = (float*)(ws + p.off_sum);
    }
}

int run_attn(const DecayParams& a, int nseg, int io_dtype, hipStream_t s) {
    if (nseg > 1) {
        if (const int e = status(launch_decay_ends(a, false, io_dtype, s))) return e;
    }
    return status(launch_decay_attn(a, io_dtype, s));
}

}  // namespace

extern "C" {

size_t triune_hip_decay_attn_workspace_size(int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv,
                                            int flags) {
    if (B <= 0 || T <= 0 || !tokens_ok(B, T) || !decay_shape_ok(H, Hk, Dk, Dv) || !seqs_ok(B, H, Dv)) return 0;
    const DecayPlan p = plan_dense(B, T, H, Dk, Dv, flags);
    return grids_ok(p, B, H, Dk, Dv) ? p.total : 0;
}

int triune_hip_decay_attn(const void* q, const void* k, const void* v, const void* g, int io_dtype, int g_dtype,
                          const int64_t* strides, float scale, const float* s0, void* o, float* s_final, int64_t B,
                          int64_t T, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv, int flags, void* workspace,
                          size_t workspace_bytes, void* stream) {
    if (!q || !k || !v || !g || !o || !strides) return TRIUNE_ERR_NULL;
    if (!dtype_ok(io_dtype) || (g_dtype != io_dtype && g_dtype != TRIUNE_DT_F32)) return TRIUNE_ERR_DTYPE;
    if (!tokens_ok(B, T) || !decay_shape_ok(H, Hk, Dk, Dv) || !seqs_ok(B, H, Dv)) return TRIUNE_ERR_SHAPE;
    if (!all_aligned(io_dtype, {q, k, v, o}) || !aligned(g, g_dtype) ||
        !all_aligned(TRIUNE_DT_F32, {s0, s_final}))
        return TRIUNE_ERR_LAYOUT;
    if (B == 0) return TRIUNE_OK;
    if (T == 0) {
        if (!s_final) return TRIUNE_OK;
        return status(launch_state_copy(s0, s_final, B * H * Dk * Dv, 4, (hipStream_t)stream));
    }
    const DecayPlan p = plan_dense(B, T, H, Dk, Dv, flags);
    if (!grids_ok(p, B, H, Dk, Dv)) return TRIUNE_ERR_SHAPE;
    if (const int e = check_ws(workspace, workspace_bytes, p.total)) return e;
    DecayParams a{};
    a.q = {q, strides[0], strides[1], strides[2]};
    a.k = {k, strides[3], strides[4], strides[5]};
    a.v = {v, strides[6], strides[7], strides[8]};
    a.g = {g, strides[9], strides[10], strides[11]};
    a.o = {o, strides[12], strides[13], strides[14]};
    a.g_dt = g_dtype, a.scale = scale, a.s0 = s0, a.fin = s_final;
    set_sizes(a, B, T, H, Hk, Dk, Dv, p, (char*)workspace);
    return run_attn(a, a.nseg, io_dtype, (hipStream_t)stream);
}

size_t triune_hip_decay_attn_varlen_workspace_size(int64_t n_seqs, int64_t total_tokens, int64_t H, int64_t Hk,
                                                   int64_t Dk, int64_t Dv, int flags) {
    if (n_seqs <= 0 || total_tokens <= 0 || !tokens_ok(n_seqs, total_tokens) || !decay_shape_ok(H, Hk, Dk, Dv) ||
        !seqs_ok(n_seqs, H, Dv))
        return 0;
    const DecayPlan p = plan_packed(n_seqs, total_tokens, H, Dk, Dv, flags);
    return grids_ok(p, n_seqs, H, Dk, Dv) ? p.total : 0;
}

int triune_hip_decay_attn_varlen(const void* q, const void* k, const void* v, const void* g, int io_dtype, int g_dtype,
                                 const int64_t* strides, float scale, const int32_t* cu_seqlens, int64_t n_seqs,
                                 int64_t total_tokens, const float* s0, float* s_final, const int32_t* slots,
                                 int64_t n_state_rows, void* o, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv,
                                 int flags, void* workspace, size_t workspace_bytes, void* stream) {
    if (!q || !k || !v || !g || !o || !strides || !cu_seqlens) return TRIUNE_ERR_NULL;
    if (!dtype_ok(io_dtype) || (g_dtype != io_dtype && g_dtype != TRIUNE_DT_F32)) return TRIUNE_ERR_DTYPE;
    if (!tokens_ok(n_seqs, total_tokens) || n_state_rows < 0 || !decay_shape_ok(H, Hk, Dk, Dv) ||
        !seqs_ok(n_seqs, H, Dv))
        return TRIUNE_ERR_SHAPE;
    if (!slots && (s0 || s_final) && n_state_rows < n_seqs) return TRIUNE_ERR_SHAPE;
    if (!all_aligned(io_dtype, {q, k, v, o}) || !aligned(g, g_dtype) ||
        !all_aligned(TRIUNE_DT_F32, {s0, s_final, cu_seqlens, slots}))
        return TRIUNE_ERR_LAYOUT;
    if (n_seqs == 0) return TRIUNE_OK;
    // with no tokens every sequence's state still passes through: one empty segment each
    const DecayPlan p = plan_packed(n_seqs, total_tokens > 0 ? total_tokens : 1, H, Dk, Dv, flags);
    if (!grids_ok(p, n_seqs, H, Dk, Dv)) return TRIUNE_ERR_SHAPE;
    if (const int e = check_ws(workspace, workspace_bytes, p.total)) return e;
    DecayParams a{};
    a.q = {q, 0, strides[0], strides[1]};
    a.k = {k, 0, strides[2], strides[3]};
    a.v = {v, 0, strides[4], strides[5]};
    a.g = {g, 0, strides[6], strides[7]};
    a.o = {o, 0, strides[8], strides[9]};
    a.g_dt = g_dtype, a.scale = scale, a.s0 = s0, a.fin = s_final;
    a.slots = slots, a.n_slots = n_state_rows, a.cu = cu_seqlens;
    set_sizes(a, n_seqs, total_tokens, H, Hk, Dk, Dv, p, (char*)workspace);
    const hipStream_t s = (hipStream_t)stream;
    if (p.nseg > 1) {
        int32_t* off = (int32_t*)((char*)workspace + p.off_seg);
        SsmParams lengths{};  // what the offsets' kernel reads of them
        lengths.cu = cu_seqlens, lengths.n_seqs = n_seqs, lengths.T = total_tokens;
        lengths.seg = (int)p.seg, lengths.n_work = p.n_work;
        if (const int e = status(launch_ssm_offsets(lengths, p.cut, off, s))) return e;
        a.seg_off = off;
    }
    return run_attn(a, a.nseg, io_dtype, s);
}

size_t triune_hip_decay_attn_bwd_workspace_size(int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv,
                                                int io_dtype, int g_head, int flags) {
    if (B <= 0 || T <= 0 || !tokens_ok(B, T) || !dtype_ok(io_dtype) || !decay_shape_ok(H, Hk, Dk, Dv) ||
        !seqs_ok(B, H, Dv))
        return 0;
    const GradPlan r = plan_grad(B, T, H, Hk, Dk, Dv, io_dtype, g_head, flags);
    return grad_grids_ok(r, B, H, Dk, Dv) ? r.total : 0;
}

int triune_hip_decay_attn_bwd(const void* q, const void* k, const void* v, const void* g, const void* dout,
                              int io_dtype, int g_dtype, const int64_t* strides, float scale, const float* s0,
                              const float* ds_final, void* dq, void* dk, void* dv, void* dg, int g_head, float* ds0,
                              int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv, int flags,
                              const void* fwd_workspace, size_t fwd_workspace_bytes, void* workspace,
                              size_t workspace_bytes, void* stream) {
    if (!q || !k || !v || !g || !dout || !strides || !dq || !dk || !dv || !dg) return TRIUNE_ERR_NULL;
    if (!dtype_ok(io_dtype) || (g_dtype != io_dtype && g_dtype != TRIUNE_DT_F32)) return TRIUNE_ERR_DTYPE;
    if (B <= 0 || T <= 0 || !tokens_ok(B, T) || !decay_shape_ok(H, Hk, Dk, Dv) || !seqs_ok(B, H, Dv))
        return TRIUNE_ERR_SHAPE;
    if (!all_aligned(io_dtype, {q, k, v, dout, dq, dk, dv}) || !aligned(g, g_dtype) || !aligned(dg, g_dtype) ||
        !all_aligned(TRIUNE_DT_F32, {s0, ds_final, ds0}))
        return TRIUNE_ERR_LAYOUT;
    const GradPlan r = plan_grad(B, T, H, Hk, Dk, Dv, io_dtype, g_head, flags);
    if (!grad_grids_ok(r, B, H, Dk, Dv)) return TRIUNE_ERR_SHAPE;
    if (fwd_workspace)
        if (const int e = check_ws(fwd_workspace, fwd_workspace_bytes, r.p.total)) return e;
    if (const int e = check_ws(workspace, workspace_bytes, fwd_workspace ? r.off_ends : r.total)) return e;
    char* ws = (char*)workspace;
    const hipStream_t s = (hipStream_t)stream;
    DecayGradParams p{};
    DecayParams& a = p.f;
    a.q = {q, strides[0], strides[1], strides[2]};
    a.k = {k, strides[3], strides[4], strides[5]};
    a.v = {v, strides[6], strides[7], strides[8]};
    a.g = {g, strides[9], strides[10], strides[11]};
    a.o = {dout, strides[12], strides[13], strides[14]};
    a.g_dt = g_dtype, a.scale = scale;
    set_sizes(a, B, T, H, Hk, Dk, Dv, r.p, ws);
    p.S = (float*)(ws + r.off_S), p.R = (float*)(ws + r.off_R);
    p.nc = r.nc, p.wide = a.slices * decay_slice((int)Dv);
    p.dq = dq, p.dk = dk, p.dv = dv, p.dg = dg;
    if (H > Hk) p.part_q = (float*)(ws + r.off_q), p.part_k = (float*)(ws + r.off_k);
    if (g_head) p.part_g = (float*)(ws + r.off_g);
    DecayWalkParams x[2];  // forward, backward
    for (const bool rev : {false, true}) {
        x[rev] = {a, (float*)(rev ? p.R : p.S), (int)r.chunk};
        DecayParams& f = x[rev].f;
        f.s0 = rev ? ds_final : s0;
        f.fin = rev ? ds0 : nullptr;
        if (rev) f.k = a.q, f.v = a.o;
        if (r.p.nseg <= 1) continue;
        f.ws_state = (float*)(!rev && fwd_workspace ? (char*)fwd_workspace : ws + (rev ? 0 : r.off_ends));
        f.ws_sum = (float*)((char*)f.ws_state + r.p.off_sum);
        if (rev || !fwd_workspace)
            if (const int e = status(launch_decay_ends(f, rev, io_dtype, s))) return e;
    }
    if (const int e = status(launch_decay_states(x[0], x[1], io_dtype, s))) return e;
    return status(launch_decay_grad(p, io_dtype, s));
}

int triune_hip_decay_attn_decode_step(const void* q, const void* k, const void* v, const void* g, int io_dtype,
                                      int g_dtype, const int64_t* strides, float scale, const float* state_in,
                                      float* state_out, const int32_t* slots, int64_t n_state_rows, void* o, int64_t B,
                                      int64_t H, int64_t Hk, int64_t Dk, int64_t Dv, void* stream) {
    if (!q || !k || !v || !g || !o || !strides || !state_in || !state_out) return TRIUNE_ERR_NULL;
    if (!dtype_ok(io_dtype) || (g_dtype != io_dtype && g_dtype != TRIUNE_DT_F32)) return TRIUNE_ERR_DTYPE;
    if (B < 0 || n_state_rows < 0 || !decay_shape_ok(H, Hk, Dk, Dv)) return TRIUNE_ERR_SHAPE;
    if (!slots && n_state_rows < B) return TRIUNE_ERR_SHAPE;
    if (!all_aligned(io_dtype, {q, k, v, o}) || !aligned(g, g_dtype) ||
        !all_aligned(TRIUNE_DT_F32, {state_in, state_out, slots}))
        return TRIUNE_ERR_LAYOUT;
    if (!grid_ok(B, H, 256)) return TRIUNE_ERR_SHAPE;
    if (B == 0) return TRIUNE_OK;
    DecayStepParams a{};
    a.q = {q, strides[0], 0, strides[1]};
    a.k = {k, strides[2], 0, strides[3]};
    a.v = {v, strides[4], 0, strides[5]};
    a.g = {g, strides[6], 0, strides[7]};
    a.o = {o, strides[8], 0, strides[9]};
    a.g_dt = g_dtype, a.scale = scale, a.s_in = state_in, a.s_out = state_out;
    a.slots = slots, a.n_rows = n_state_rows, a.Bn = B;
    a.H = (int)H, a.per = (int)(H / Hk), a.Dk = (int)Dk, a.Dv = (int)Dv;
    return status(launch_decay_step(a, io_dtype, (hipStream_t)stream));
}

// ---- norms ---------------------------------------------------------------------------------------
static int rms_check(std::initializer_list<const void*> io, const void* w, const void* s, int io_dtype, int w_dtype,
                     int s_dtype, int64_t R, int64_t G, int64_t D) {
    auto par_ok = [&](const void* p, int dt) { return !p || dt == io_dtype || dt == TRIUNE_DT_F32; };
    if (!dtype_ok(io_dtype) || !par_ok(w, w_dtype) || !par_ok(s, s_dtype)) return TRIUNE_ERR_DTYPE;
    if (R < 0 || R > kMaxGrid || G <= 0 || G > kMaxGrid || D <= 0 || D > NORM_MAX_D) return TRIUNE_ERR_SHAPE;
    if (!all_aligned(io_dtype, io) || !aligned(w, w_dtype) || !aligned(s, s_dtype)) return TRIUNE_ERR_LAYOUT;
    return TRIUNE_OK;
}

int triune_hip_rms_norm(const void* x, const void* r, const void* w, const void* s, int io_dtype, int r_dtype,
                        int w_dtype, int s_dtype, const int64_t* strides, float alpha, float eps, void* y, void* h,
                        float* rstd, int64_t R, int64_t G, int64_t D, void* stream) {
    if (!x || !y || !strides || (r == nullptr) != (h == nullptr)) return TRIUNE_ERR_NULL;
    if (const int e = rms_check({x, y}, w, s, io_dtype, w_dtype, s_dtype, R, G, D)) return e;
    if (r && r_dtype != io_dtype && r_dtype != TRIUNE_DT_F32) return TRIUNE_ERR_DTYPE;
    if ((r && !all_aligned(r_dtype, {r, h})) || !aligned(rstd, TRIUNE_DT_F32)) return TRIUNE_ERR_LAYOUT;
    if (R == 0) return TRIUNE_OK;
    RmsParams a{};
    a.x = {x, strides[0], strides[1]};
    a.r = {r, strides[2], strides[3]};
    a.w = w, a.s = s, a.w_dt = w_dtype, a.s_dt = s_dtype, a.alpha = alpha, a.eps = eps;
    a.y = y, a.h = h, a.rstd = rstd, a.R = R, a.G = (int)G, a.D = (int)D, a.cus = compute_units();
    return status(launch_rms_norm(a, io_dtype, r && r_dtype != io_dtype, (hipStream_t)stream));
}

size_t triune_hip_rms_norm_bwd_workspace_size(int64_t R, int64_t D) {
    if (R <= 0 || R > kMaxGrid || D <= 0 || D > NORM_MAX_D) return 0;
    return align_up((size_t)rms_bwd_parts(R, (int)D, compute_units()) * 2 * D * 4);
}

static int rms_parts(RmsBwdParams& p, void* ws, size_t have) {
    p.parts = rms_bwd_parts(p.f.R, p.f.D, p.f.cus);
    if (!p.dw && !p.ds) return TRIUNE_OK;
    p.part = (float*)ws;
    return check_ws(ws, have, (size_t)p.parts * 2 * p.f.D * 4);
}

int triune_hip_rms_norm_bwd(const void* h, const void* dy, const void* dh, const void* x, const void* w,
                            const void* s, int io_dtype, int h_dtype, int w_dtype, int s_dtype, const int64_t* strides,
                            float alpha, const float* rstd, void* dx, void* dr, void* dw, void* ds, int64_t R,
                            int64_t G, int64_t D, void* workspace, size_t workspace_bytes, void* stream) {
    if (!h || !dy || !rstd || !strides || (ds && (!x || !s))) return TRIUNE_ERR_NULL;
    if (const int e = rms_check({dy, x, dx}, w, s, io_dtype, w_dtype, s_dtype, R, G, D)) return e;
    if (h_dtype != io_dtype && h_dtype != TRIUNE_DT_F32) return TRIUNE_ERR_DTYPE;
    if (!all_aligned(h_dtype, {h, dh, dr}) || !aligned(rstd, TRIUNE_DT_F32) || !aligned(dw, w_dtype) ||
        !aligned(ds, s_dtype))
        return TRIUNE_ERR_LAYOUT;
    if (R == 0) return TRIUNE_ERR_SHAPE;
    RmsBwdParams p{};
    RmsParams& a = p.f;
    a.r = {h, strides[0], strides[1]};
    p.dy = {dy, strides[2], strides[3]};
    p.dh = {dh, strides[4], strides[5]};
    a.x = {x, strides[6], strides[7]};
    a.w = w, a.s = s, a.w_dt = w_dtype, a.s_dt = s_dtype, a.alpha = alpha, a.rstd = const_cast<float*>(rstd);
    a.R = R, a.G = (int)G, a.D = (int)D, a.cus = compute_units();
    p.dx = dx, p.dr = dr, p.dw = dw, p.ds = ds;
    if (const int e = rms_parts(p, workspace, workspace_bytes)) return e;
    return status(launch_rms_norm_bwd(p, io_dtype, h_dtype != io_dtype, (hipStream_t)stream));
}

int triune_hip_gated_rms_norm(const void* x, const void* z, const void* w, int io_dtype, int w_dtype,
                              const int64_t* strides, float eps, void* y, float* rstd, int64_t R, int64_t G, int64_t D,
                              void* stream) {
    if (!x || !z || !y || !strides) return TRIUNE_ERR_NULL;
    if (const int e = rms_check({x, z, y}, w, nullptr, io_dtype, w_dtype, 0, R, G, D)) return e;
    if (!aligned(rstd, TRIUNE_DT_F32)) return TRIUNE_ERR_LAYOUT;
    if (R == 0) return TRIUNE_OK;
    RmsParams a{};
    a.x = {x, strides[0], strides[1]};
    a.z = {z, strides[2], strides[3]};
    a.w = w, a.w_dt = w_dtype, a.eps = eps, a.y = y, a.rstd = rstd;
    a.R = R, a.G = (int)G, a.D = (int)D, a.cus = compute_units();
    return status(launch_gated_norm(a, io_dtype, (hipStream_t)stream));
}

int triune_hip_gated_rms_norm_bwd(const void* x, const void* z, const void* dy, const void* w, int io_dtype,
                                  int w_dtype, const int64_t* strides, const float* rstd, void* dx, void* dz, void* dw,
                                  int64_t R, int64_t G, int64_t D, void* workspace, size_t workspace_bytes,
                                  void* stream) {
    if (!x || !z || !dy || !rstd || !strides) return TRIUNE_ERR_NULL;
    if (const int e = rms_check({x, z, dy, dx, dz}, w, nullptr, io_dtype, w_dtype, 0, R, G, D)) return e;
    if (!aligned(rstd, TRIUNE_DT_F32) || !aligned(dw, w_dtype)) return TRIUNE_ERR_LAYOUT;
    if (R == 0) return TRIUNE_ERR_SHAPE;
    RmsBwdParams p{};
    RmsParams& a = p.f;
    a.x = {x, strides[0], strides[1]};
    a.z = {z, strides[2], strides[3]};
    p.dy = {dy, strides[4], strides[5]};
    a.w = w, a.w_dt = w_dtype, a.rstd = const_cast<float*>(rstd);
    a.R = R, a.G = (int)G, a.D = (int)D, a.cus = compute_units();
    p.dx = dx, p.dz = dz, p.dw = dw;
    if (const int e = rms_parts(p, workspace, workspace_bytes)) return e;
    return status(launch_gated_norm_bwd(p, io_dtype, (hipStream_t)stream));
}

}  // extern "C"
