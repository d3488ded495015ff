"""GPU: the selective scan against its 64-bit definition (ssm_ref.py): prompts, packed prompts, single
tokens, gradients, and the calls' refusals."""

import pytest
import torch
import ssm_ref as R

from triune_amd import ssm as S
from triune_amd import ssm_decode_step, ssm_scan, ssm_scan_varlen

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def inputs(dev, B, T, D, N, G=1, dtype=F32, z=True, skip=True, bias=True, s0=True, seed=0, slow=False):
    """u, delta, A, B, C and keywords, on the device.  slow: steps of 1e-3 and less, long memories."""
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    bc = (B, T, N) if G == 1 else (B, T, G, N)
    to = lambda x: x.to(dtype).to(dev)  # noqa: E731
    args = [to(rn(B, T, D)), to(rn(B, T, D)), (-torch.exp(0.7 * rn(D, N))).to(dev), to(rn(*bc)), to(rn(*bc))]
    kw = {"D": rn(D).to(dev) if skip else None, "z": to(rn(B, T, D)) if z else None,
          "delta_bias": ((rn(D) - 7) if slow else rn(D)).to(dev) if bias else None,
          "initial_state": rn(B, D, N).to(dev) if s0 else None}
    return args, kw


def want(args, kw, soft=True):
    return R.scan(*args, kw["D"], kw["z"], kw["delta_bias"], soft, kw["initial_state"])


def check(got, ref, dtype, what=""):
    R.near(got[0], ref[0], ref[2], dtype, f"{what} y")
    R.near(got[1], ref[1], ref[3], F32, f"{what} state")


SHAPES = [  # B, T, D, N, G
    (1, 1, 1, 1, 1), (2, 5, 3, 2, 1), (1, 31, 64, 4, 1), (2, 32, 65, 5, 1), (1, 33, 130, 16, 1), (2, 100, 96, 16, 2),
    (1, 257, 40, 24, 1), (1, 70, 70, 40, 1), (2, 40, 33, 64, 3), (1, 64, 128, 8, 2), (3, 17, 200, 12, 1),
]


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("shape", SHAPES)
def test_scan(dev, shape, dtype):
    B, T, D, N, G = shape
    args, kw = inputs(dev, B, T, D, N, G, dtype, seed=T)
    check(ssm_scan(*args, **kw), want(args, kw), dtype)


@pytest.mark.parametrize("z", [True, False])
@pytest.mark.parametrize("skip", [True, False])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("s0", [True, False])
@pytest.mark.parametrize("soft", [True, False])
def test_scan_optional_parts(dev, z, skip, bias, s0, soft):
    args, kw = inputs(dev, 2, 40, 70, 16, z=z, skip=skip, bias=bias, s0=s0, seed=5)
    if not soft:
        args[1] = args[1].abs() * 0.1
        kw["delta_bias"] = kw["delta_bias"].abs() * 0.1 if bias else None
    check(ssm_scan(*args, delta_softplus=soft, **kw), want(args, kw, soft), F32)


@pytest.mark.parametrize("units", [1, 2, 3])
@pytest.mark.parametrize("shape", [(2, 200, 70, 16, 1), (1, 161, 96, 24, 2), (1, 64, 20, 3, 1), (1, 97, 64, 50, 1)])
def test_scan_in_segments(dev, units, shape):
    """Segments of 32, 64 and 96 tokens, whatever length the rule would take."""
    B, T, D, N, G = shape
    args, kw = inputs(dev, B, T, D, N, G, seed=T)
    y, s, _ = S._scan(*args, kw["D"], kw["z"], kw["delta_bias"], True, kw["initial_state"], None, False, units << 8)
    check((y, s), want(args, kw), F32)


def test_long_memory(dev):
    """4096 tokens with steps near 1e-3: states hold thousands of tokens, and the rule splits the time
    axis; in float32 and against the unsplit call."""
    args, kw = inputs(dev, 1, 4096, 40, 16, slow=True, seed=9)
    got = ssm_scan(*args, **kw)
    assert S.plan_on(args[0], "triune_hip_ssm_scan_workspace_size", 1, 4096, 40, 1, 16, 0) > 0
    check(got, want(args, kw), F32)


def test_strides_and_broadcasts(dev):
    """Views of projections, transposed batches, inputs broadcast along the batch and along time, odd
    element offsets, an output buffer of strided rows."""
    args, kw = inputs(dev, 2, 50, 66, 10, seed=2, dtype=BF)
    ref = want(args, kw)
    u, delta, A, B, C = args
    wide = torch.zeros(2, 50, 200, device=dev, dtype=BF)
    wide[..., 1:67], wide[..., 67:133] = u, kw["z"]
    proj = torch.zeros(50, 2, 33, device=dev, dtype=BF)
    proj[..., 3:13], proj[..., 13:23] = B.transpose(0, 1), C.transpose(0, 1)
    proj = proj.transpose(0, 1)
    buf = torch.full((2, 50, 70), 7.0, device=dev, dtype=BF)
    k2 = {**kw, "z": wide[..., 67:133], "out": buf[..., 2:68]}
    y, s = ssm_scan(wide[..., 1:67], delta.transpose(1, 2).contiguous().transpose(1, 2), A.t().contiguous().t(),
                    proj[..., 3:13], proj[..., 13:23], **k2)
    assert y.data_ptr() == buf[..., 2:68].data_ptr()
    check((y, s), ref, BF)
    assert bool((buf[..., :2] == 7).all()) and bool((buf[..., 68:] == 7).all())
    # the same row for the whole batch, and one token for all times
    b1 = [args[0][:1].expand(2, -1, -1), args[1][:, :1].expand(-1, 50, -1), A, B[:1, :1].expand(2, 50, -1), C]
    check(ssm_scan(*b1, **kw), want(b1, kw), BF)


def test_extremes(dev):
    """Steps that decay everything, steps of zero, A of zero, an infinite step: no NaN comes of them."""
    args, kw = inputs(dev, 1, 40, 64, 16, s0=True, bias=False, seed=3)
    args[1][:, 5] = 90.0
    args[1][:, 9] = -200.0
    args[1][:, 11] = -1e30
    args[2][:, 0] = 0.0
    args[2][:, 1] = -1e4
    kw["z"][:, 3] = 120.0
    kw["z"][:, 4] = -120.0
    check(ssm_scan(*args, **kw), want(args, kw), F32)


def test_masked_tokens(dev):
    """delta of -inf or of the type's lowest value is a step of 0 (the state stays, and gradients), one
    near the largest forgets all."""
    for dtype in (F32, BF):
        args, kw = inputs(dev, 2, 70, 68, 16, dtype=dtype, seed=21)
        args[1][:, 3] = args[1][:, 64] = float("-inf")
        args[1][:, 4] = args[1][1, 40:] = torch.finfo(dtype).min
        args[1][:, 20], args[0][:, 20] = 2e38, 0.0
        check(ssm_scan(*args, **kw), want(args, kw), dtype)
        x = [t[:, 3] if t.dim() == 3 else t for t in args]
        k = {**kw, "z": kw["z"][:, 3]}
        s0 = k.pop("initial_state")
        assert torch.equal(ssm_decode_step(*x, s0, **k)[1], s0)
    args[1][:, 20] = 1.0
    leaves = [t.requires_grad_() for t in args]
    y, s = ssm_scan(*leaves, **kw)
    grads = torch.autograd.grad(y.float().sum() + s.sum(), leaves)
    assert all(bool(t.isfinite().all()) for t in grads)
    assert bool((grads[1][:, [3, 4, 64]] == 0).all()) and bool((grads[3][:, [3, 4, 64]] == 0).all())


def test_nan_stays_in_its_row(dev):
    """A NaN of one batch row, channel or later token reaches no other row, channel or earlier token."""
    args, kw = inputs(dev, 3, 70, 70, 16, seed=4)
    ref = [t.clone() for t in ssm_scan(*args, **kw)]
    args[0][1, 40, 69] = float("nan")
    y, s = ssm_scan(*args, **kw)
    assert bool(y[1, 40:, 69].isnan().all()) and bool(s[1, 69].isnan().all())
    y[1, 40:, 69], s[1, 69] = ref[0][1, 40:, 69], ref[1][1, 69]
    assert torch.equal(y, ref[0]) and torch.equal(s, ref[1])


def test_empty(dev):
    args, kw = inputs(dev, 2, 0, 8, 4)
    y, s = ssm_scan(*args, **kw)
    assert y.shape == (2, 0, 8) and torch.equal(s, kw["initial_state"])
    args, kw = inputs(dev, 0, 4, 8, 4)
    y, s = ssm_scan(*args, **kw)
    assert y.shape == (0, 4, 8) and s.shape == (0, 8, 4)


def test_empty_gradients(dev):
    """No tokens: the initial state's gradient is the final state's, every other gradient is zero."""
    args, kw = inputs(dev, 2, 0, 8, 4)
    leaves = [t.requires_grad_() for t in (*args, *kw.values())]
    y, s = ssm_scan(*args, **kw)
    got = torch.autograd.grad((y.sum(), s.sum()), leaves)
    for x, g in zip(leaves, got):
        assert g.shape == x.shape and bool((g == (1 if x is kw["initial_state"] else 0)).all())


# ---- packed ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("lens", [[1], [5, 0, 33, 1, 64, 100], [0, 0], [300, 2], [3] * 70])
@pytest.mark.parametrize("G", [1, 2])
def test_varlen_matches_each_sequence(dev, lens, G):
    D, N = 72, 12
    total, n = sum(lens) + 9, len(lens)  # nine rows before and behind the sequences
    args, kw = inputs(dev, 1, total, D, N, G, seed=n)
    s0 = torch.randn(n, D, N, generator=torch.Generator().manual_seed(1)).to(dev)
    cu = torch.tensor([4] + lens, dtype=torch.int32).cumsum(0).to(torch.int32)
    out = torch.full((1, total, D), 7.0, device=dev)
    k2 = {**kw, "initial_state": s0}
    y, s = ssm_scan_varlen(*args, cu, out=out, **k2)
    assert y.data_ptr() == out.data_ptr()
    assert bool((y[0, :4] == 7).all()) and bool((y[0, int(cu[-1]):] == 7).all())
    for i, ln in enumerate(lens):
        c = slice(int(cu[i]), int(cu[i]) + ln)
        part = [args[0][:, c], args[1][:, c], args[2], args[3][:, c], args[4][:, c]]
        ref = R.scan(*part, kw["D"], kw["z"][:, c], kw["delta_bias"], True, s0[i:i + 1])
        check((y[:, c], s[i:i + 1]), ref, F32, f"sequence {i}")


def test_varlen_in_many_segments(dev):
    """A long sequence among short ones: the rule splits it."""
    lens, D, N = [1500, 1, 70], 64, 16
    args, kw = inputs(dev, 1, sum(lens), D, N, seed=8)
    assert S.plan_on(args[0], "triune_hip_ssm_scan_varlen_workspace_size", 3, sum(lens), D, 1, N, 0) > 0
    cu = torch.tensor([0, 1500, 1501, 1571], device=dev)
    kw["initial_state"] = None
    y, s = ssm_scan_varlen(*args, cu, **kw)
    for i, ln in enumerate(lens):
        c = slice(int(cu[i]), int(cu[i]) + ln)
        part = [args[0][:, c], args[1][:, c], args[2], args[3][:, c], args[4][:, c]]
        check((y[:, c], s[i:i + 1]), R.scan(*part, kw["D"], kw["z"][:, c], kw["delta_bias"], True, None), F32)


@pytest.mark.parametrize("long", [False, True])
def test_varlen_pool(dev, long):
    """Slots of a pool in place, in any order; a slot outside the pool keeps nothing, other rows stay."""
    lens = [40, 900 if long else 3, 0, 7]
    D, N = 64, 16
    args, kw = inputs(dev, 1, sum(lens), D, N, seed=6)
    flat = [args[0][0], args[1][0], args[2], args[3][0], args[4][0]]
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(dev)
    pool = torch.randn(6, D, N, generator=torch.Generator().manual_seed(2)).to(dev)
    before = pool.clone()
    slots = torch.tensor([4, 0, 2, -1], device=dev, dtype=torch.int32)
    y, p = ssm_scan_varlen(*flat, cu, D=kw["D"], z=kw["z"][0], delta_bias=kw["delta_bias"], state_pool=pool,
                           slots=slots)
    assert p is pool
    for i, ln in enumerate(lens):
        c, sl = slice(int(cu[i]), int(cu[i]) + ln), int(slots[i])
        part = [args[0][:, c], args[1][:, c], args[2], args[3][:, c], args[4][:, c]]
        ref = R.scan(*part, kw["D"], kw["z"][:, c], kw["delta_bias"], True, before[sl:sl + 1] if sl >= 0 else None)
        R.near(y[None, c], ref[0], ref[2], F32, f"sequence {i}")
        if sl >= 0:
            R.near(pool[sl:sl + 1], ref[1], ref[3], F32, f"slot {sl}")
    for r in (1, 2, 3, 5):
        assert torch.equal(pool[r], before[r])


# ---- single tokens --------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (3, 70, 16, 1), (2, 96, 5, 2), (5, 64, 64, 1), (2, 33, 24, 3), (4, 50, 8, 1)])
def test_decode_step(dev, shape, dtype):
    B, D, N, G = shape
    args, kw = inputs(dev, B, 1, D, N, G, dtype, seed=D)
    state = kw.pop("initial_state")
    ref = R.scan(*args, kw["D"], kw["z"], kw["delta_bias"], True, state)
    keep = state.clone()
    y, s = ssm_decode_step(*args, state, **kw)
    assert torch.equal(state, keep)
    check((y, s), ref, dtype)
    flat = [args[0][:, 0], args[1][:, 0], args[2], args[3][:, 0], args[4][:, 0]]
    kw["z"] = kw["z"][:, 0]
    y2, s2 = ssm_decode_step(*flat, state, inplace=True, **kw)
    assert s2 is state and torch.equal(s2, s) and torch.equal(y2, y[:, 0])


def test_decode_slots(dev):
    args, kw = inputs(dev, 4, 1, 70, 16, seed=1)
    kw.pop("initial_state")
    pool = torch.randn(6, 70, 16, device=dev)
    before = pool.clone()
    slots = torch.tensor([5, -1, 0, 6], device=dev)
    ref = R.scan(*args, kw["D"], kw["z"], kw["delta_bias"], True, before[[5, 0, 0, 0]])
    y, p = ssm_decode_step(*args, pool, slots=slots, inplace=True, **kw)
    for b, sl in ((0, 5), (2, 0)):
        R.near(y[b], ref[0][b], ref[2][b], F32)
        R.near(pool[sl], ref[1][b], ref[3][b], F32)
    assert bool((y[1] == 0).all()) and bool((y[3] == 0).all())
    assert torch.equal(pool[1:5], before[1:5])
    new, np_ = ssm_decode_step(*args, before, slots=slots, **kw)
    assert torch.equal(new, y) and torch.equal(np_, pool) and np_ is not before


def test_prompt_then_tokens_is_one_prompt(dev):
    args, kw = inputs(dev, 2, 45, 70, 16, seed=7)
    y, s = ssm_scan(*args, **kw)
    a = [x if x.dim() == 2 else x[:, :41] for x in args]
    k = {**kw, "z": kw["z"][:, :41]}
    y1, st = ssm_scan(*a, **k)
    ref = want(args, kw)
    outs = [y1]
    for t in range(41, 45):
        c = slice(t, t + 1)
        yt, st = ssm_decode_step(args[0][:, c], args[1][:, c], args[2], args[3][:, c], args[4][:, c], st, D=kw["D"],
                                 z=kw["z"][:, c], delta_bias=kw["delta_bias"], inplace=True)
        outs.append(yt)
    check((torch.cat(outs, 1), st), ref, F32)
    check((y, s), ref, F32)


# ---- gradients ------------------------------------------------------------------------------------
NAMES = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "initial_state")


def grad_check(dev, args, kw, dtype, soft=True, flags=None, use_y=True, use_s=True):
    """The operator's gradients against the formulas: every term carries at most 24 (T + 16) units, T
    tokens' decays and states forward and T backward with at most 12 roundings each."""
    B, T, D = args[0].shape
    N = args[2].shape[1]
    g = torch.Generator().manual_seed(11)
    dy = torch.randn(B, T, D, generator=g).to(dtype).to(dev) if use_y else None
    ds = torch.randn(B, D, N, generator=g).to(dev) if use_s else None
    leaves = [t.clone().requires_grad_() if t is not None else None
              for t in (*args, kw["D"], kw["z"], kw["delta_bias"], kw["initial_state"])]
    live = [t for t in leaves if t is not None]
    if flags is None:
        y, s = ssm_scan(*leaves[:5], D=leaves[5], z=leaves[6], delta_bias=leaves[7], delta_softplus=soft,
                        initial_state=leaves[8])
        outs = [(o, d) for o, d in ((y, dy), (s, ds)) if d is not None]
        got = dict(zip(map(id, live), torch.autograd.grad([o for o, _ in outs], live, [d for _, d in outs])))
        got = [None if t is None else got[id(t)] for t in leaves]
    else:
        p = [None if t is None else t.detach() for t in leaves]
        _, _, kept = S._scan(*p[:8], soft, p[8], None, True, flags)
        got = S._scan_bwd(*p[:8], soft, kept, dy, ds, p[8] is not None, flags)
    zero = torch.zeros(B, T, D)
    form = [*args, kw["D"], kw["z"], kw["delta_bias"], soft, kw["initial_state"], zero if dy is None else dy, ds]
    ref, env = R.scan_grads(*form), R.scan_grads(*form, absolute=True)
    for name, x, r, e in zip(NAMES, got, ref, env):
        if r is None:
            assert x is None, name
            continue
        io = dtype if name in ("u", "delta", "B", "C", "z") else F32
        assert x.dtype == io
        R.near(x, r, 24 * (T + 16) * R.U * e, io, name)
    return got


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("shape", SHAPES)
def test_gradients(dev, shape, dtype):
    B, T, D, N, G = shape
    args, kw = inputs(dev, B, T, D, N, G, dtype, seed=T + 1)
    grad_check(dev, args, kw, dtype)


@pytest.mark.parametrize("z,skip,bias,s0,soft", [
    (False, True, True, True, True), (True, False, True, True, True), (True, True, False, True, True),
    (True, True, True, False, True), (True, True, True, True, False), (False, False, False, False, False)])
def test_gradients_optional_parts(dev, z, skip, bias, s0, soft):
    args, kw = inputs(dev, 2, 40, 70, 16, z=z, skip=skip, bias=bias, s0=s0, seed=5)
    if not soft:
        args[1] = args[1].abs() * 0.1
        kw["delta_bias"] = kw["delta_bias"].abs() * 0.1 if bias else None
    grad_check(dev, args, kw, F32, soft)


@pytest.mark.parametrize("use_y,use_s", [(True, False), (False, True)])
def test_gradients_of_one_output(dev, use_y, use_s):
    args, kw = inputs(dev, 2, 40, 70, 16, seed=5)
    grad_check(dev, args, kw, F32, use_y=use_y, use_s=use_s)


@pytest.mark.parametrize("units", [1, 2])
@pytest.mark.parametrize("shape", [(2, 200, 70, 16, 1), (1, 161, 96, 24, 2), (1, 97, 64, 50, 1), (1, 70, 20, 3, 1)])
def test_gradients_in_segments(dev, units, shape):
    B, T, D, N, G = shape
    args, kw = inputs(dev, B, T, D, N, G, seed=T)
    grad_check(dev, args, kw, F32, flags=units << 8)


def test_gradients_of_broadcast_inputs(dev):
    """B and C shared over the batch, u over time: their gradients are the sums over what they were
    broadcast to."""
    args, kw = inputs(dev, 2, 40, 66, 16, seed=5)
    u, B, C = args[0][:, :1].clone().requires_grad_(), args[3][:1].clone().requires_grad_(), args[4][:1].clone().requires_grad_()
    full = [u.expand(-1, 40, -1), args[1], args[2], B.expand(2, -1, -1), C.expand(2, -1, -1)]
    y, _ = ssm_scan(*full, **kw)
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(1)).to(dev)
    got = torch.autograd.grad(y, (u, B, C), dy)
    form = [*(t.detach() for t in full), kw["D"], kw["z"], kw["delta_bias"], True, kw["initial_state"], dy, None]
    ref, env = R.scan_grads(*form), R.scan_grads(*form, absolute=True)
    for x, k, dim in zip(got, (0, 3, 4), (1, 0, 0)):
        R.near(x, ref[k].sum(dim, keepdim=True), 24 * 57 * R.U * env[k].sum(dim, keepdim=True), F32)


def test_only_some_inputs_need_gradients(dev):
    args, kw = inputs(dev, 1, 20, 64, 16, seed=5)
    args[2].requires_grad_()
    y, s = ssm_scan(*args, **kw)
    (dA,) = torch.autograd.grad(y.sum() + s.sum(), args[2])
    assert dA.shape == (64, 16) and bool(dA.isfinite().all())
    with pytest.raises(RuntimeError):  # once differentiable
        y, _ = ssm_scan(*args, **kw)
        (g,) = torch.autograd.grad(y.sum(), args[2], create_graph=True)
        g.sum().backward()


def test_results_do_not_depend_on_timing(dev):
    args, kw = inputs(dev, 2, 333, 200, 16, seed=5, dtype=BF)
    a = grad_check(dev, args, kw, BF)
    b = grad_check(dev, args, kw, BF)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


# ---- streams, graphs, refusals ------------------------------------------------------------------------
def test_another_stream(dev):
    args, kw = inputs(dev, 2, 300, 64, 16, seed=5)
    ref = ssm_scan(*args, **kw)
    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = ssm_scan(*args, **kw)
    torch.cuda.current_stream(dev).wait_stream(side)
    for x, y in zip(got, ref):
        assert torch.equal(x, y)


def test_two_graphs_with_segments(dev):
    """Two captured calls with workspaces of their own, replayed in turn with eager work between."""
    sets = [inputs(dev, 1, 600, 40, 16, seed=s) for s in (1, 2)]
    cu = torch.tensor([0, 50, 600], device=dev, dtype=torch.int32)
    eager = [[t.clone() for t in ssm_scan(*a, **k)] for a, k in sets]
    graphs = []
    for a, k in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ssm_scan(*a, **k)
            kv = {**k, "initial_state": None}
            packed = ssm_scan_varlen(*a, cu, **kv)
        graphs.append((g, out, packed))
    ev = [ssm_scan_varlen(*a, cu, **{**k, "initial_state": None}) for a, k in sets]
    for r in range(3):
        for (g, out, packed), want_, pv, (a, k) in zip(graphs, eager, ev, sets):
            for t in (*out, *packed):
                t.fill_(float("nan"))
            g.replay()
            ssm_scan(*a, **k)
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, want_))
            assert all(torch.equal(x, y) for x, y in zip(packed, pv))


def test_backward_replays_from_a_graph(dev):
    args, kw = inputs(dev, 2, 200, 70, 16, seed=3, dtype=BF)
    p = [*args, kw["D"], kw["z"], kw["delta_bias"]]
    _, _, kept = S._scan(*p, True, kw["initial_state"], None, True)
    dy, ds = torch.randn_like(args[0]), torch.randn(2, 70, 16, device=dev)
    call = lambda: S._scan_bwd(*p, True, kept, dy, ds, True)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for n in range(3):
        dy.copy_(torch.randn(dy.shape, generator=torch.Generator().manual_seed(n)))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip([t.clone() for t in out], call()):
            assert torch.equal(x, y)


def test_decode_replays_from_a_graph(dev):
    args, kw = inputs(dev, 4, 1, 70, 16, seed=1)
    kw.pop("initial_state")
    pool = torch.zeros(6, 70, 16, device=dev)
    slots = torch.tensor([5, 1, 0, 3], device=dev, dtype=torch.int32)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, _ = ssm_decode_step(*args, pool, slots=slots, inplace=True, **kw)
    other = pool.zero_().clone()
    for n in range(3):
        args[0].copy_(torch.randn(args[0].shape, generator=torch.Generator().manual_seed(n)))
        g.replay()
        e, _ = ssm_decode_step(*args, other, slots=slots, inplace=True, **kw)
        torch.cuda.synchronize()
        assert torch.equal(y, e) and torch.equal(pool, other)


def test_refusals(dev):
    args, kw = inputs(dev, 2, 8, 8, 4)
    u, delta, A, B, C = args
    bad = [
        (dict(a=[u[0], delta, A, B, C]), ValueError), (dict(a=[u, delta[:, :4], A, B, C]), ValueError),
        (dict(a=[u, delta, A[:4], B, C]), ValueError), (dict(a=[u, delta, A.bfloat16(), B, C]), TypeError),
        (dict(a=[u, delta, A, B[..., :2], C]), ValueError), (dict(a=[u, delta, A, B.bfloat16(), C]), TypeError),
        (dict(a=[u.double(), delta, A, B, C]), TypeError), (dict(a=[u, delta, A.cpu(), B, C]), ValueError),
        (dict(z=u[:1]), ValueError), (dict(z=u.half()), TypeError), (dict(D=kw["D"][:4]), ValueError),
        (dict(delta_bias=kw["D"].half()), TypeError), (dict(initial_state=kw["initial_state"][:1]), ValueError),
        (dict(out=torch.empty(2, 8, 8, device=dev, dtype=BF)), ValueError),
        (dict(out=torch.empty(2, 8, 9, device=dev)[..., :8].transpose(1, 2)), ValueError),
        (dict(out=torch.empty(2, 1, 8, device=dev).expand(2, 8, 8)), ValueError),
        (dict(a=[u, delta, torch.zeros(8, 65, device=dev), torch.zeros(2, 8, 65, device=dev),
                 torch.zeros(2, 8, 65, device=dev)]), ValueError),
        (dict(a=[u, delta, A, torch.zeros(2, 8, 3, 4, device=dev), torch.zeros(2, 8, 3, 4, device=dev)]), ValueError),
    ]
    for change, err in bad:
        a = change.pop("a", args)
        with pytest.raises(err):
            ssm_scan(*a, **{**kw, **change})
    with pytest.raises(ValueError, match="gradient"):
        ssm_scan(u, delta, A.clone().requires_grad_(), B, C, out=torch.empty_like(u))
    cu = torch.tensor([0, 8], device=dev, dtype=torch.int32)
    one = [t if t.dim() == 2 else t[:1] for t in args]
    pool = torch.zeros(3, 8, 4, device=dev)
    sl = torch.zeros(1, device=dev, dtype=torch.int32)
    with pytest.raises(ValueError, match="gradient"):
        ssm_scan_varlen(one[0], one[1], A.clone().requires_grad_(), *one[3:], cu)
    for k in (dict(state_pool=pool), dict(state_pool=pool.half(), slots=sl), dict(slots=sl),
              dict(state_pool=pool, slots=sl[:0]), dict(state_pool=pool[:, :4], slots=sl),
              dict(state_pool=pool, slots=sl, initial_state=pool[:1]), dict(initial_state=pool)):
        with pytest.raises(ValueError):
            ssm_scan_varlen(*one, cu, **k)
    with pytest.raises(ValueError):
        ssm_scan_varlen(*args, cu)  # batch of two
    with pytest.raises(ValueError):
        ssm_scan_varlen(*one, cu.float())
    with pytest.raises(ValueError):
        ssm_decode_step(*args, pool)  # eight tokens
    step = [t if t.dim() == 2 else t[:, 0] for t in args]
    for k in (dict(), dict(slots=sl), dict(slots=torch.zeros(2, 1, device=dev))):
        with pytest.raises(ValueError):
            ssm_decode_step(*step, pool, **k)
    with pytest.raises(ValueError):
        ssm_decode_step(*step, pool[:2].half(), inplace=True)
    with pytest.raises(ValueError):
        ssm_decode_step(*step, pool.transpose(1, 2)[:2])


def test_pools_that_want_gradients_are_refused(dev):
    """A pool is written in place, without a gradient."""
    args, kw = inputs(dev, 1, 8, 8, 4)
    packed = [t[0] if t.dim() == 3 else t for t in args]
    cu, slots = torch.tensor([0, 8], dtype=torch.int32, device=dev), torch.tensor([0], dtype=torch.int32, device=dev)
    pool = torch.zeros(2, 8, 4, device=dev, requires_grad=True)
    with pytest.raises(ValueError):
        ssm_scan_varlen(*packed, cu, state_pool=pool, slots=slots)
    with torch.no_grad():
        assert ssm_scan_varlen(*packed, cu, state_pool=pool, slots=slots)[1] is pool


def test_more_segments_than_a_block_joins_at_once(dev):
    """139 segments of 32 tokens with long memories, forward and gradients, and a packed call whose one long prompt
    has more segments than the average that the join is laid out for."""
    args, kw = inputs(dev, 1, 4430, 10, 5, slow=True, seed=31)
    y, s, _ = S._scan(*args, kw["D"], kw["z"], kw["delta_bias"], True, kw["initial_state"], None, False, 1 << 8)
    check((y, s), want(args, kw), F32)
    grad_check(dev, args, kw, F32, flags=1 << 8)
    lens = [3, 4400, *[1] * 26, 1]
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(dev)
    s0 = kw["initial_state"].expand(len(lens), -1, -1)
    kw["initial_state"] = None
    yp, fin = ssm_scan_varlen(*args, cu, **{**kw, "initial_state": s0})
    for i in (0, 1, len(lens) - 1):
        c = slice(int(cu[i]), int(cu[i + 1]))
        part = [args[0][:, c], args[1][:, c], args[2], args[3][:, c], args[4][:, c]]
        check((yp[:, c], fin[i:i + 1]), R.scan(*part, kw["D"], kw["z"][:, c], kw["delta_bias"], True, s0[:1]), F32)
