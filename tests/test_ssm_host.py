"""CPU: what the state space layer's entry points refuse before anything is launched."""

import ctypes

import pytest
import torch

import triune_amd
import triune_amd._lib as L

FAKE = ctypes.c_void_p(0x1000)  # aligned, never read: validation fails first or there is nothing to do
ODD = ctypes.c_void_p(0x1001)
NULL, SHAPE, DTYPE, LAYOUT, WORKSPACE = -1, -2, -3, -4, -5


def st(n):
    return (ctypes.c_int64 * n)(*([64] * n))


def caller(name, order, **base):
    fn = getattr(L.lib(), name)

    def call(**kw):
        a = {**base, **kw}
        return fn(*[a[k] for k in order])

    return call


SCAN = "u dl z B C A D bias io st soft s0 y fin kept Bn T Dm G N flags ws wsb stream".split()
VARLEN = "u dl z B C A D bias io st soft cu n total s0 fin slots rows y Dm G N flags ws wsb stream".split()
BWD = ("u dl z B C A D bias dy io st soft kept dfin du dd dz dB dC dA dD db ds0 Bn T Dm G N flags ws wsb "
       "stream").split()
STEP = "u dl z B C A D bias io st soft s_in s_out slots rows y Bn Dm G N stream".split()


def _scan_base(names):
    base = {k: FAKE for k in names}
    base.update(io=1, st=st(14), soft=1, z=None, D=None, bias=None, slots=None, ws=None, wsb=0, stream=None, flags=0,
                Bn=2, T=64, Dm=64, G=1, N=16, n=2, total=64, rows=2, dz=None)
    return base


@pytest.mark.parametrize("name,order", [("triune_hip_ssm_scan", SCAN), ("triune_hip_ssm_scan_varlen", VARLEN),
                                        ("triune_hip_ssm_bwd", BWD), ("triune_hip_ssm_decode_step", STEP)])
def test_scan_entries_refuse(name, order):
    call = caller(name, order, **_scan_base(order))
    for k in ("u", "dl", "B", "C", "A", "st"):
        assert call(**{k: None}) == NULL
    assert call(io=7) == DTYPE
    for kw in ({"N": 0}, {"N": 65}, {"G": 0}, {"G": 3}, {"Dm": 0}, {"Dm": 1 << 28}):
        assert call(**kw) == SHAPE, kw
    for k in ("u", "dl", "B", "C", "A", "D", "bias"):
        assert call(**{k: ODD}) == LAYOUT, k
    if "T" in order:
        assert call(T=-1) == SHAPE and call(T=1 << 30) == SHAPE and call(Bn=-1) == SHAPE
        assert call(Bn=1 << 40, T=1 << 29) == SHAPE  # more workgroups than a grid holds
    if "rows" in order:
        assert call(rows=1) == SHAPE  # fewer state rows than sequences and no slots
        assert call(slots=ODD) == LAYOUT
    if "cu" in order:
        assert call(cu=None) == NULL and call(cu=ODD) == LAYOUT and call(total=-1) == SHAPE


def test_scan_entries_need_their_workspace():
    call = caller("triune_hip_ssm_bwd", BWD, **_scan_base(BWD))
    need = L.lib().triune_hip_ssm_bwd_workspace_size(2, 64, 64, 1, 16, 0)
    assert need > 0
    assert call(ws=None, wsb=need) == WORKSPACE and call(ws=FAKE, wsb=need - 1) == WORKSPACE
    assert call(ws=ctypes.c_void_p(0x1004), wsb=need) == LAYOUT
    for k in ("kept", "du", "dd", "dB", "dC", "dA", "dy"):
        assert call(**{k: None}) == NULL, k
    assert call(z=FAKE) == NULL  # a gate without its gradient
    assert call(Bn=0) == SHAPE and call(T=0) == SHAPE
    scan = caller("triune_hip_ssm_scan", SCAN, **_scan_base(SCAN))
    flags = 1 << 8  # segments of 32 tokens
    need = L.lib().triune_hip_ssm_scan_workspace_size(2, 64, 64, 1, 16, flags)
    assert need >= 2 * 2 * 17 * 64 * 4
    assert scan(flags=flags, ws=FAKE, wsb=need - 1) == WORKSPACE


def test_empty_calls_launch_nothing():
    assert caller("triune_hip_ssm_scan", SCAN, **_scan_base(SCAN))(T=0) == 0
    assert caller("triune_hip_ssm_scan", SCAN, **_scan_base(SCAN))(Bn=0) == 0
    assert caller("triune_hip_ssm_scan_varlen", VARLEN, **_scan_base(VARLEN))(n=0) == 0
    assert caller("triune_hip_ssm_decode_step", STEP, **_scan_base(STEP))(Bn=0) == 0
    assert L.lib().triune_hip_ssm_scan_workspace_size(0, 64, 64, 1, 16, 0) == 0


CONV = "x w bias io wdt st silu s0 fin y Bn T Dm W stream".split()
CONV_V = "x w bias io wdt st silu cu n total s0 fin slots rows y Dm W stream".split()
CONV_S = "x w bias io wdt st silu s0 fin slots rows y Bn Dm W stream".split()
CONV_B = "x w bias dy io wdt st silu s0 dfin dx dw db ds0 Bn T Dm W ws wsb stream".split()


def _conv_base(names):
    base = {k: FAKE for k in names}
    base.update(io=1, wdt=1, st=st(4), silu=1, bias=None, slots=None, ws=None, wsb=0, stream=None, Bn=2, T=64, Dm=64, W=4,
                n=2, total=64, rows=2)
    return base


@pytest.mark.parametrize("name,order", [
    ("triune_hip_short_conv", CONV), ("triune_hip_short_conv_varlen", CONV_V),
    ("triune_hip_short_conv_decode_step", CONV_S), ("triune_hip_short_conv_bwd", CONV_B)])
def test_conv_entries_refuse(name, order):
    call = caller(name, order, **_conv_base(order))
    for k in ("x", "w", "st"):
        assert call(**{k: None}) == NULL
    assert call(io=7) == DTYPE and call(wdt=2) == DTYPE and call(io=0, wdt=1) == DTYPE
    for kw in ({"W": 1}, {"W": 5}, {"Dm": 0}, {"Dm": 1 << 28}):
        assert call(**kw) == SHAPE, kw
    for k in ("x", "w", "bias", "s0"):
        assert call(**{k: ODD}) == LAYOUT, k
    if "rows" in order:
        assert call(rows=1) == SHAPE and call(slots=ODD) == LAYOUT
    if "T" in order:
        assert call(T=1 << 30) == SHAPE and call(Bn=1 << 24, T=1 << 20) == SHAPE
    if "cu" in order:
        assert call(cu=None) == NULL and call(cu=ODD) == LAYOUT
    if "ws" in order:
        need = L.lib().triune_hip_short_conv_bwd_workspace_size(2, 64, 64, 4)
        assert need > 0 and call(ws=FAKE, wsb=need - 1) == WORKSPACE and call(dy=None) == NULL


NORM = "x xs w b io wdt bdt eps y mean rstd R D stream".split()
NORM_B = "x xs w dy ys io wdt bdt mean rstd dx dw db R D ws wsb stream".split()


def test_norm_entries_refuse():
    base = dict(x=FAKE, xs=64, w=FAKE, b=FAKE, io=1, wdt=1, bdt=0, eps=1e-5, y=FAKE, mean=None, rstd=None, R=4, D=64,
                stream=None, dy=FAKE, ys=64, dx=FAKE, dw=FAKE, db=FAKE, ws=None, wsb=0)
    fwd = caller("triune_hip_layer_norm", NORM, **base)
    bwd = caller("triune_hip_layer_norm_bwd", NORM_B, **{**base, "mean": FAKE, "rstd": FAKE})
    for call in (fwd, bwd):
        assert call(x=None) == NULL and call(io=5) == DTYPE and call(wdt=2) == DTYPE and call(bdt=2) == DTYPE
        assert call(D=0) == SHAPE and call(D=16385) == SHAPE and call(R=-1) == SHAPE
        assert call(x=ODD) == LAYOUT and call(w=ODD) == LAYOUT
    assert fwd(y=None) == NULL and fwd(mean=FAKE) == NULL and fwd(R=0) == 0
    need = L.lib().triune_hip_layer_norm_bwd_workspace_size(4, 64)
    assert need > 0 and bwd(ws=FAKE, wsb=need - 1) == WORKSPACE and bwd(R=0) == SHAPE and bwd(dx=None) == NULL


def test_operators_refuse_cpu_tensors():
    x, w = torch.zeros(1, 4, 8), torch.zeros(8, 4)
    with pytest.raises(ValueError, match="CPU"):
        triune_amd.short_conv(x, w)
    with pytest.raises(ValueError, match="CPU"):
        triune_amd.layer_norm(x)
    with pytest.raises(ValueError, match="CPU"):
        triune_amd.ssm_scan(x, x, w, torch.zeros(1, 4, 4), torch.zeros(1, 4, 4))


def test_counts_past_the_plans_numbers():
    """Counts whose products with channels or tokens pass 64 bits are refused, not multiplied."""
    lib, many = L.lib(), 1 << 60
    for call in (caller("triune_hip_ssm_scan", SCAN, **_scan_base(SCAN)),
                 caller("triune_hip_ssm_bwd", BWD, **_scan_base(BWD)),
                 caller("triune_hip_short_conv", CONV, **_conv_base(CONV)),
                 caller("triune_hip_short_conv_bwd", CONV_B, **_conv_base(CONV_B))):
        assert call(Bn=many) == SHAPE
    for call in (caller("triune_hip_ssm_scan_varlen", VARLEN, **_scan_base(VARLEN)),
                 caller("triune_hip_short_conv_varlen", CONV_V, **_conv_base(CONV_V))):
        assert call(n=many, rows=many) == SHAPE
    assert lib.triune_hip_ssm_scan_workspace_size(many, 64, 64, 1, 16, 0) == 0
    assert lib.triune_hip_ssm_bwd_workspace_size(many, 64, 64, 1, 16, 0) == 0
    assert lib.triune_hip_ssm_scan_varlen_workspace_size(many, 64, 64, 1, 16, 0) == 0
    assert lib.triune_hip_short_conv_bwd_workspace_size(many, 64, 64, 4) == 0


def test_forward_mode_duals_are_refused():
    """What every entry asks of its tensors: no tangent, recorded or not."""
    fw, x = torch.autograd.forward_ad, torch.zeros(3)
    from triune_amd.ssm import _needs_grad

    assert not _needs_grad(x, None)
    with fw.dual_level():
        assert not _needs_grad(x, None) and _needs_grad(None, torch.zeros(3, requires_grad=True))
        d = fw.make_dual(x, torch.ones(3))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="forward-mode"):
                _needs_grad(None, x, d)
    assert not _needs_grad(x)


def test_out_rows_that_overlap():
    """Rows of two dims on one another, though each stride spans a row; interleaved rows are apart."""
    from triune_amd.ssm import _out

    flat, like = torch.zeros(256), torch.zeros(1)
    for st in ((8, 8, 1), (16, 8, 1), (56, 8, 1), (8, 12, 1), (64, 4, 1), (64, 8, 2), (0, 8, 1)):
        with pytest.raises(ValueError, match="overlap"):
            _out(flat.as_strided((2, 8, 8), st), (2, 8, 8), torch.float32, like, 1)
    for st in ((64, 8, 1), (8, 16, 1), (9, 18, 1), (100, 10, 1)):
        _out(flat.as_strided((2, 8, 8), st), (2, 8, 8), torch.float32, like, 1)
    for shape, st in (((1, 8, 8), (0, 8, 1)), ((2, 1, 8), (8, 0, 1)), ((2, 8, 1), (8, 1, 5)), ((0, 8, 8), (0, 0, 1))):
        _out(flat.as_strided(shape, st), shape, torch.float32, like, 1)


def test_slots_past_32_bits():
    from triune_amd.ssm import _slots

    dev, wide = torch.device("cpu"), [3, 0, -1, -7, (1 << 32) + 1, -(1 << 32), 1 << 31, -(1 << 31) - 1]
    got = _slots(torch.tensor(wide), len(wide), dev)
    assert got.dtype == torch.int32
    for s, g in zip(wide, got.tolist()):
        assert g == s if 0 <= s < 1 << 31 else g < 0 or g == (1 << 31) - 1  # stays outside every pool
    for dt in (torch.int8, torch.int16, torch.uint8, torch.int32):
        assert _slots(torch.tensor([3, 0], dtype=dt), 2, dev).tolist() == [3, 0]
    for dt in (torch.float32, torch.float16, torch.bool, torch.complex64, torch.uint64, torch.uint32):
        with pytest.raises(TypeError, match="slots"):
            _slots(torch.zeros(2, dtype=dt), 2, dev)


def test_tokens_wider_than_the_kernels_address():
    """2^22 group states a token and more: refused by name, and not copied first; one token has no stride."""
    from triune_amd.ssm import _rows

    B = torch.zeros(1).expand(1, 2, 1 << 16, 64)
    with pytest.raises(ValueError, match="too wide"):
        _rows(B, 1)
    with pytest.raises(ValueError, match="too wide"):
        _rows(B[0], 0)
    assert _rows(B[:, :1, :4], 1).shape == (1, 1, 4, 64) and _rows(B[:, :, : (1 << 16) - 1, :8], 1).is_contiguous()


def test_grids_past_32_bits_of_threads():
    """Channel groups of one channel make a workgroup each, sixteen waves above 32 states: 2^32 threads are refused,
    not launched."""
    wide = dict(st=(ctypes.c_int64 * 14)(*([4096] * 14)), T=1, total=1024, n=1024, Bn=1024, rows=1024, Dm=4096, G=4096,
                N=64)
    big, ws = L.lib().triune_hip_ssm_bwd_workspace_size(1024, 1, 4096, 4096, 64, 0), FAKE
    assert caller("triune_hip_ssm_scan", SCAN, **{**_scan_base(SCAN), **wide})() == SHAPE
    assert caller("triune_hip_ssm_scan_varlen", VARLEN, **{**_scan_base(VARLEN), **wide})() == SHAPE
    assert caller("triune_hip_ssm_bwd", BWD, **{**_scan_base(BWD), **wide})(ws=ws, wsb=big) == SHAPE


@pytest.mark.parametrize("N,split,whole", [
    (16, [256, 304], [320, 352, 448, 504, 512]), (8, [512], [640, 768]), (32, [128], [160, 192]),
    (64, [64, 128], [160, 192])])
def test_scans_are_split_where_that_is_faster(N, split, whole):
    """Workgroups (8 prompts of 2048 tokens) on both sides of the measured crossover."""
    size = L.lib().triune_hip_ssm_scan_workspace_size
    for wgs in split:
        assert size(8, 2048, wgs * 8, 1, N, 0) > 0, wgs
    for wgs in whole:
        assert size(8, 2048, wgs * 8, 1, N, 0) == 0, wgs


@pytest.mark.parametrize("N,split,whole", [
    (16, [256, 320, 400], [448, 504, 512]), (8, [512, 640], [832, 1024]), (32, [128, 160, 192], [208, 240]),
    (64, [64, 128, 160], [192, 240])])
def test_gradients_are_split_where_that_is_faster(N, split, whole):
    size, unsplit = L.lib().triune_hip_ssm_bwd_workspace_size, 255 << 8
    for wgs in split:
        assert size(8, 2048, wgs * 8, 1, N, 0) > size(8, 2048, wgs * 8, 1, N, unsplit), wgs
    for wgs in whole:
        assert size(8, 2048, wgs * 8, 1, N, 0) == size(8, 2048, wgs * 8, 1, N, unsplit), wgs


def test_packed_scans_with_one_long_prompt_are_cut():
    """Sequences enough for two rounds of the chip: 42 of 64 tokens and one of 16384 (1536 channels) have room for
    segments, calls of few tokens have none and need none."""
    size = L.lib().triune_hip_ssm_scan_varlen_workspace_size
    assert size(43, 42 * 64 + 16384, 1536, 1, 16, 0) > 43 * 17 * 1536 * 4
    assert size(201, 28000, 1536, 1, 16, 0) > 201 * 17 * 1536 * 4
    assert size(100, 3000, 1536, 1, 16, 0) == 0 and size(43, 43, 1536, 1, 16, 0) == 0


def test_packed_scans_of_thousands_of_sequences_are_taken():
    """The join's grid counts what it launches: blocks for the segments that are followed, of the waves they get."""
    call = caller("triune_hip_ssm_scan_varlen", VARLEN, **_scan_base(VARLEN))
    for n, total, Dm, N in ((4200, 8400, 1088, 64), (4096, 200000, 4096, 16), (20000, 40000, 768, 64)):
        need = L.lib().triune_hip_ssm_scan_varlen_workspace_size(n, total, Dm, 1, N, 0)
        kw = dict(n=n, rows=n, total=total, Dm=Dm, N=N, st=(ctypes.c_int64 * 8)(*([Dm] * 8)))
        assert need > 0 and call(ws=FAKE, wsb=need - 1, **kw) == WORKSPACE, (n, total, Dm, N)


def test_offsets_past_32_bits():
    """int64 offsets stay on their side of the packed rows, to which the kernels cut them."""
    from triune_amd.ssm import _cu

    dev = torch.device("cpu")
    got = _cu(torch.tensor([-(1 << 32) + 3, 0, 7, (1 << 32) + 5]), dev)
    assert got.dtype == torch.int32 and got.tolist() == [0, 0, 7, (1 << 31) - 1]
    assert _cu(torch.tensor([0, 7], dtype=torch.int32), dev).tolist() == [0, 7]
