"""CPU: what the decay attention layer's entry points refuse before anything is launched."""

import ctypes

import pytest
import torch
from test_ssm_host import DTYPE, FAKE, LAYOUT, NULL, ODD, SHAPE, WORKSPACE, caller, st

import triune_amd
import triune_amd._lib as L
from triune_amd import decay as A
from triune_amd import norm as N

DENSE = "q k v g io gdt st scale s0 o fin B T H Hk Dk Dv flags ws wsb stream".split()
VARLEN = "q k v g io gdt st scale cu n total s0 fin slots rows o H Hk Dk Dv flags ws wsb stream".split()
BWD = "q k v g do io gdt st scale s0 dfin dq dk dv dg head ds0 B T H Hk Dk Dv flags fws fwsb ws wsb stream".split()
STEP = "q k v g io gdt st scale s_in s_out slots rows o B H Hk Dk Dv stream".split()
ENTRIES = [("triune_hip_decay_attn", DENSE), ("triune_hip_decay_attn_varlen", VARLEN),
           ("triune_hip_decay_attn_bwd", BWD), ("triune_hip_decay_attn_decode_step", STEP)]


def base(names, **kw):
    b = {k: FAKE for k in names}
    b.update(io=1, gdt=0, st=st(15), scale=1.0, slots=None, ws=None, wsb=0, stream=None, flags=0, B=2, T=64, H=4, Hk=2,
             Dk=64, Dv=64, n=2, total=64, rows=2, head=0, fws=None, fwsb=0)
    return {**b, **kw}


@pytest.mark.parametrize("name,order", ENTRIES)
def test_attention_entries_refuse(name, order):
    call = caller(name, order, **base(order))
    for k in ("q", "k", "v", "g", "st"):
        assert call(**{k: None}) == NULL
    assert call(io=7) == DTYPE and call(gdt=2) == DTYPE
    for kw in ({"Dk": 0}, {"Dk": 129}, {"Dv": 0}, {"Dv": 16385}, {"H": 0}, {"Hk": 0}, {"Hk": 3}, {"H": 1 << 16, "Hk": 1}):
        assert call(**kw) == SHAPE, kw
    for k in ("q", "k", "v", "g"):
        assert call(**{k: ODD}) == LAYOUT, k
    if "B" in order:
        assert call(B=-1) == SHAPE and call(B=1 << 60, rows=1 << 60) == SHAPE and call(B=1 << 30, rows=1 << 30) == SHAPE
    if "T" in order:
        assert call(T=-1) == SHAPE and call(T=1 << 30) == SHAPE
    if "rows" in order:
        assert call(rows=1) == SHAPE and call(slots=ODD) == LAYOUT  # fewer state rows than sequences and no slots
    if "cu" in order:
        assert call(cu=None) == NULL and call(cu=ODD) == LAYOUT and call(total=-1) == SHAPE
        assert call(n=1 << 60, rows=1 << 60) == SHAPE and call(n=1 << 30, rows=1 << 30) == SHAPE


def test_attention_entries_need_their_workspace():
    lib = L.lib()
    need = lib.triune_hip_decay_attn_bwd_workspace_size(2, 64, 4, 2, 64, 64, 1, 0, 0)
    call = caller("triune_hip_decay_attn_bwd", BWD, **base(BWD))
    assert need >= 2 * 2 * 4 * 64 * 64 * 4 + 2 * 2 * 64 * 4 * 64 * 4
    assert call(ws=None, wsb=need) == WORKSPACE and call(ws=FAKE, wsb=need - 1) == WORKSPACE
    assert call(ws=ctypes.c_void_p(0x1004), wsb=need) == LAYOUT
    for k in ("do", "dq", "dk", "dv", "dg"):
        assert call(**{k: None}) == NULL, k
    assert call(B=0) == SHAPE and call(T=0) == SHAPE
    flags = 1 << 8  # segments of 64 tokens (packed: 32)
    need = lib.triune_hip_decay_attn_workspace_size(2, 128, 4, 2, 64, 64, flags)
    assert need >= 2 * 2 * 4 * 64 * 64 * 4
    dense = caller("triune_hip_decay_attn", DENSE, **base(DENSE))
    assert dense(T=128, flags=flags, ws=FAKE, wsb=need - 1) == WORKSPACE
    assert call(T=128, flags=flags, fws=FAKE, fwsb=need - 1, ws=FAKE, wsb=1 << 40) == WORKSPACE
    need = lib.triune_hip_decay_attn_varlen_workspace_size(2, 640, 4, 2, 64, 64, flags)
    varlen = caller("triune_hip_decay_attn_varlen", VARLEN, **base(VARLEN))
    assert need > 0 and varlen(flags=flags, total=640, ws=FAKE, wsb=need - 1) == WORKSPACE
    for many in (1 << 60, 1 << 30):
        assert lib.triune_hip_decay_attn_workspace_size(many, 64, 4, 2, 64, 64, 0) == 0
        assert lib.triune_hip_decay_attn_bwd_workspace_size(many, 64, 4, 2, 64, 64, 1, 0, 0) == 0
        assert lib.triune_hip_decay_attn_varlen_workspace_size(many, 64, 4, 2, 64, 64, 0) == 0


def test_empty_calls_launch_nothing():
    assert caller("triune_hip_decay_attn", DENSE, **base(DENSE))(B=0) == 0
    assert caller("triune_hip_decay_attn", DENSE, **base(DENSE))(T=0, fin=None) == 0
    assert caller("triune_hip_decay_attn_varlen", VARLEN, **base(VARLEN))(n=0) == 0
    assert caller("triune_hip_decay_attn_decode_step", STEP, **base(STEP))(B=0) == 0


RMS = "x r w s io rdt wdt sdt st alpha eps y h rstd R G D stream".split()
RMS_B = "h dy dh x w s io rdt wdt sdt st alpha rstd dx dr dw ds R G D ws wsb stream".split()
GATED = "x z w io wdt st eps y rstd R G D stream".split()
GATED_B = "x z dy w io wdt st rstd dx dz dw R G D ws wsb stream".split()


def test_norm_entries_refuse():
    b = {k: FAKE for k in {*RMS, *RMS_B, *GATED, *GATED_B}}
    b.update(io=1, rdt=0, wdt=1, sdt=0, st=st(8), alpha=1.0, eps=1e-6, R=4, G=1, D=64, ws=None, wsb=0, stream=None)
    rms, rms_b = caller("triune_hip_rms_norm", RMS, **b), caller("triune_hip_rms_norm_bwd", RMS_B, **b)
    gated, gated_b = caller("triune_hip_gated_rms_norm", GATED, **b), caller("triune_hip_gated_rms_norm_bwd", GATED_B, **b)
    for call, must in ((rms, "x y"), (rms_b, "h dy rstd"), (gated, "x z y"), (gated_b, "x z dy rstd")):
        for k in (*must.split(), "st"):
            assert call(**{k: None}) == NULL, k
        assert call(io=5) == DTYPE and call(wdt=2) == DTYPE and call(w=ODD) == LAYOUT and call(rstd=ODD) == LAYOUT
        assert call(D=0) == SHAPE and call(D=16385) == SHAPE and call(R=-1) == SHAPE and call(R=1 << 31) == SHAPE
        assert call(G=0) == SHAPE
        for k in must.split()[:2]:
            assert call(**{k: ODD}) == LAYOUT, k
    assert rms(R=0) == 0 and gated(R=0) == 0 and rms_b(R=0) == SHAPE and gated_b(R=0) == SHAPE
    assert rms(rdt=2) == DTYPE and rms(sdt=2) == DTYPE and rms(h=None) == NULL and rms(r=None) == NULL
    assert rms_b(rdt=2) == DTYPE and rms_b(x=None) == NULL and rms_b(s=None) == NULL
    need = L.lib().triune_hip_rms_norm_bwd_workspace_size(4, 64)
    for call in (rms_b, gated_b):
        assert need > 0 and call(ws=FAKE, wsb=511) == WORKSPACE and call(ws=ctypes.c_void_p(0x1004), wsb=need) == LAYOUT
    assert L.lib().triune_hip_rms_norm_bwd_workspace_size(0, 64) == 0


def test_operators_refuse_cpu_tensors():
    x, g = torch.zeros(1, 4, 2, 8), torch.zeros(1, 4, 2)
    for call in (lambda: triune_amd.decay_attn(x, x, x, g), lambda: triune_amd.rms_norm(x),
                 lambda: triune_amd.decay_attn_varlen(x, x, x, g, torch.tensor([0, 4])),
                 lambda: triune_amd.decay_attn_decode_step(x[:, :1], x[:, :1], x[:, :1], g[:, :1], x),
                 lambda: triune_amd.add_rms_norm(x, x), lambda: triune_amd.gated_rms_norm(x, x)):
        with pytest.raises(ValueError, match="CPU"):
            call()


def test_head_strides():
    assert A._head_strides(torch.zeros(2, 3, 4, 5)) == (60, 20, 5)
    assert A._head_strides(torch.zeros(2, 3, 4), 3) == (12, 4, 1)
    assert A._head_strides(torch.zeros(8)[::2], 3) == (0, 0, 2) and A._head_strides(torch.zeros(4), 2) == (0, 1)


def test_rows_of_two_strides():
    """Rows of one outer and one inner stride go as they are, others are copied."""
    x = torch.zeros(4, 6, 5, 16)
    for v, want in ((x, (80, 16)), (x[:, :, 1:4], (80, 16)), (x[..., :8], (80, 16)), (x[0], (80, 16)), (x[0, 0], (16, 16)),
                    (x[0, 0, 0], (16, 16)), (x[:1, ::2], (160, 16)), (x[:, 0], (480, 16))):
        got, outer, inner = N._pair(v, N._inner(v))
        assert got is v and (outer, inner) == want, v.shape
    for v in (x[:, 1:3], x.transpose(-1, -2), x[..., ::2], x[:1].expand(3, 6, 5, 16)):
        got, outer, inner = N._pair(v, N._inner(v))
        assert got.is_contiguous() and got.shape == v.shape and inner == v.shape[-1] and outer == v.shape[-2] * inner


def test_segments_by_length_and_heads():
    """Dense calls are cut where their (sequence, head) pairs leave the card idle, and nowhere else."""
    size = L.lib().triune_hip_decay_attn_workspace_size

    def segments(B, T, H, Dk, Dv, values, flags=0):
        """Segments of a sequence, from the states and sums that a workspace holds."""
        have = size(B, T, H, H, Dk, Dv, flags)
        pad = lambda n: -(-n // 256) * 256  # noqa: E731
        return next((n for n in range(2, T // 64 + 2)
                     if have == pad(4 * B * n * H * values) + pad(8 * B * n * H)), 1 if have == 0 else None)

    for T in (1, 63, 64):
        assert segments(1, T, 1, 64, 64, 64 * 64) == 1, T
    for T in (65, 127, 128):
        assert segments(1, T, 1, 64, 64, 64 * 64) in (1, 2), T
    assert segments(1, 640, 1, 64, 64, 64 * 64) == 10  # never shorter than 64 tokens
    assert segments(1, 640, 1, 128, 300, 128 * 384) == 10  # value dims in whole slices
    assert segments(1, 640, 1, 64, 64, 64 * 64, 4 << 8) == 5  # forced: of 4 x 32 tokens
    assert segments(1 << 12, 640, 16, 64, 64, 64 * 64) == 1  # workgroups enough
    assert size(1, 640, 1, 1, 0, 64, 0) == 0 and size(0, 640, 1, 1, 64, 64, 0) == 0
