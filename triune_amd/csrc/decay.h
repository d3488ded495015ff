// decay.h -- parameter blocks and launchers of the decay attention kernels (decay_attn.hip, decay_walk.hip,
// decay_attn_bwd.hip).  Internal to libtriune_hip.
#pragma once

#include "ssm.h"

namespace triune {

constexpr int DECAY_MAX_DK = 128, DECAY_MAX_DV = 16384;
constexpr int DECAY_CHUNK = 32;

// A [tokens, heads, dim] operand of a batch of sequences: element strides, innermost stride 1.  A gate has no dim.
struct DecayTok {
    const void* p;
    int64_t sb, st, sh;
};

struct DecayParams {
    DecayTok q, k, v, g, o;
    int g_dt;
    float scale;
    const float* s0;          // [rows, H, Dk, Dv] or null
    float* fin;               // [rows, H, Dk, Dv] or null
    const int32_t* slots;     // packed over a pool: the row of each sequence, else null
    int64_t n_slots;
    float* ws_state;          // [n_work, H, values]: a segment's own end state, then the state behind it; the last
                              // segment's place: the sequence's initial state
    float* ws_sum;            // [n_work, H, 2]: summed log2 decays
    int64_t n_seqs, T;        // T: length of a dense sequence, or all tokens of a packed call
    int H, per, Dk, Dv;       // per: heads of v for one of q and k
    int slices;               // column slices of the state
    int seg, nseg;            // tokens of a segment, segments of a dense sequence
    int64_t n_work;
    const int32_t *cu, *seg_off;  // packed: [n_seqs + 1] token and segment offsets
};

// Columns of a slice, and the values that a segment's state takes in the workspace.
int decay_slice(int Dv);
int decay_padded_dk(int Dk);
int64_t decay_state_values(int Dk, int Dv);
// Whether the rows of these tensors are whole 16-byte units (for fp16, eight bytes), aligned, and 32 of them within the
// offsets of a buffer resource.
inline bool decay_full(int Dk, int Dv, int io_dt, std::initializer_list<DecayTok> ts) {
    const int e = io_dt == DT_BF16 ? 8 : 4, size = io_dt == DT_F32 ? 4 : 2;
    if (Dk % e || Dv % e) return false;
    for (const DecayTok& t : ts) {
        if (!t.p) continue;
        if (reinterpret_cast<uintptr_t>(t.p) % (e * size) || (t.sb | t.st | t.sh) & (e - 1)) return false;
        if (t.st < 0 || t.st >= (TILE_SKIP >> 8)) return false;  // 63 rows of 4 bytes and a row's width stay below it
    }
    return true;
}

// Segments' end states and what the join makes of them, in the workspace; rev: gradients of states, from the end.
hipError_t launch_decay_ends(const DecayParams& a, bool rev, int io_dt, hipStream_t s);

// The states in front of every chunk, and the gradients of those behind them.
struct DecayWalkParams {
    DecayParams f;            // rows in k, columns in v
    float* states;            // [n_seqs, H, nc, DK, columns], nc = ceil(T / every)
    int every;                // a multiple of 32 tokens; segments are multiples of it
};
hipError_t launch_decay_states(const DecayWalkParams& states, const DecayWalkParams& grads, int io_dt, hipStream_t s);
hipError_t launch_decay_attn(const DecayParams& a, int io_dt, hipStream_t s);

// Tokens of a chunk of the gradients: 64, or 32 for operands in fp32, whose tiles take twice the LDS.
constexpr int decay_grad_chunk(bool bf16) { return bf16 ? 64 : 32; }

struct DecayGradParams {
    DecayParams f;            // o: the gradient of the outputs
    const float *S, *R;       // states in front of the chunks, gradients of those behind them (DecayWalkParams)
    int64_t wide;             // columns of a state as kept
    int64_t nc;               // chunks of a sequence
    void *dq, *dk, *dv;       // contiguous, I/O dtype
    float *part_q, *part_k;   // [n_seqs T, H, Dk] where heads share q and k, else null
    void* dg;                 // [n_seqs, T, H], or [H] with part_g
    float* part_g;            // [n_seqs nc, H] or null
};
hipError_t launch_decay_grad(const DecayGradParams& p, int io_dt, hipStream_t s);

struct DecayStepParams {
    DecayTok q, k, v, g, o;   // sb and sh: strides of the batch and the heads
    int g_dt;
    float scale;
    const float* s_in;
    float* s_out;
    const int32_t* slots;
    int64_t n_rows, Bn;
    int H, per, Dk, Dv;
};
hipError_t launch_decay_step(const DecayStepParams& a, int io_dt, hipStream_t s);

// ---- device helpers --------------------------------------------------------------------------
// A log-decay in units of the hardware's exp2: above 0 it counts as 0, below -512 (a factor of 0 even for the
// largest state) as -512; NaN stays.
__device__ __forceinline__ float log2_gate(float g) {
    const float x = g * LOG2E;
    return x > 0.f ? 0.f : x < -512.f ? -512.f : x;
}
__device__ __forceinline__ float load_dt(const void* p, int dt, int64_t i) {
    if (dt == DT_F32) return ((const float*)p)[i];
    if (dt == DT_BF16) return (float)((const __bf16*)p)[i];
    return (float)((const _Float16*)p)[i];
}

// Sums of log-decays as hi + lo: hi is a multiple of 2^-8, so sums of it are exact up to 2^16, and |lo| stays
// small, so the difference of two sums is as exact as its own size and not theirs (a token that forgets all
// leaves sums of hundreds, behind which decays of 1e-3 still count).
struct Sum2 {
    float hi, lo;
};
__device__ __forceinline__ Sum2 split_gate(float x) {
    const float hi = __builtin_rintf(x * 256.f) * (1.f / 256.f);
    return {hi, x - hi};
}
__device__ __forceinline__ float decay_between(const Sum2& a, const Sum2& b) {  // 2^(a - b)
    return __builtin_amdgcn_exp2f((a.hi - b.hi) + (a.lo - b.lo));
}

}  // namespace triune
