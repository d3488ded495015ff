"""GPU: corners of the state space layer's operators that their other tests leave."""

import ctypes

import pytest
import torch
import ssm_ref as R

import triune_amd._lib as L
from triune_amd import (layer_norm, short_conv, short_conv_decode_step, short_conv_varlen, ssm_decode_step, ssm_scan,
                        ssm_scan_varlen)
from triune_amd import ssm as S

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


# ---- modes that grow --------------------------------------------------------------------------------
# dt A = 2 a token: 92 binary exponents in 32 tokens, 185 in 64, past the largest number's 128.
def growing(dev, B, T, D=40, N=16, seed=0):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    u, Bm, C = rn(B, T, D), rn(B, T, N), rn(B, T, N)
    A = torch.full((D, N), 2.0) - 0.1 * torch.rand(D, N, generator=g)
    A[:, 1] = -1.0  # beside them one that decays
    return [t.to(dev) for t in (u, torch.ones(B, T, D), A, Bm, C)]


def growing_check(got, args, s0=None):
    y, fin, ey, ef, _ = R.scan(*args, soft=False, s0=s0)
    R.near(got[0], y, ey, F32, "y")
    R.near(got[1], fin, ef, F32, "state")


@pytest.mark.parametrize("units", [0, 1, 2, 3])
def test_zero_states_grow_to_zero(dev, units):
    """Left padding (u = 0, no initial state) in front of 12 tokens: the state stays 0 whatever its decay product is,
    so the split call gives what the unsplit one does."""
    args = growing(dev, 2, 212)
    args[0][:, :200] = 0
    y, s, _ = S._scan(*args, None, None, None, False, None, None, False, units << 8)
    growing_check((y, s), args)


def test_zero_states_grow_to_zero_by_the_rule(dev):
    """The same through the public calls, where the rule splits the time axis: dense and packed."""
    args = growing(dev, 1, 4096)
    args[0][:, :4084] = 0
    assert S.plan_on(args[0], "triune_hip_ssm_scan_workspace_size", 1, 4096, 40, 1, 16, 0) > 0
    growing_check(ssm_scan(*args, delta_softplus=False), args)
    lens = [300, 3784, 12]
    args[0][:, 288:300] = args[0][:, 4080:4084] = 1
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(dev)
    assert S.plan_on(args[0], "triune_hip_ssm_scan_varlen_workspace_size", 3, 4096, 40, 1, 16, 0) > 0
    y, s = ssm_scan_varlen(*args, cu, delta_softplus=False)
    for i, ln in enumerate(lens):
        c = slice(int(cu[i]), int(cu[i]) + ln)
        growing_check((y[:, c], s[i:i + 1]), [t if t.dim() == 2 else t[:, c] for t in args])


@pytest.mark.parametrize("units", [0, 1, 2])
def test_small_states_grow_within_range(dev, units):
    """A state of 1e-30 grows by 2^207 to about 2^107, though the decay product of its first 64 tokens is past the
    largest number; a large one decays by 2^-200 to a small one."""
    args = growing(dev, 1, 72, seed=1)
    args[0].zero_()
    s0 = torch.full((1, 40, 16), 1e-30, device=dev)
    args[2][:, 1], s0[:, :, 1] = -2.0, 1e30
    y, s, _ = S._scan(*args, None, None, None, False, s0, None, False, units << 8)
    growing_check((y, s), args, s0)


@pytest.mark.parametrize("units", [0, 1, 2])
def test_gradients_of_growing_modes(dev, units):
    """Upstream of the first 12 tokens only: the gradient of every later state is 0 whatever it is decayed by."""
    args = growing(dev, 2, 212, seed=2)
    args[0][:, :200] = 0
    s0 = torch.zeros(2, 40, 16, device=dev)
    dy = torch.randn(2, 212, 40, generator=torch.Generator().manual_seed(3)).to(dev)
    dy[:, 12:] = 0
    _, _, kept = S._scan(*args, None, None, None, False, s0, None, True, units << 8)
    got = S._scan_bwd(*args, None, None, None, False, kept, dy, None, True, units << 8)
    form = (*args, None, None, None, False, s0, dy, None)
    for x, r, e in zip(got, R.scan_grads(*form), R.scan_grads(*form, absolute=True)):
        assert (x is None) == (r is None)
        if r is not None:
            R.near(x, r, 24 * (212 + 16) * R.U * e, F32)


# ---- infinite decays ----------------------------------------------------------------------------------
@pytest.mark.parametrize("soft", [True, False])
@pytest.mark.parametrize("N", [3, 16, 40])
def test_gradients_with_infinite_decay(dev, N, soft):
    """A of -inf forgets at every step above 0, as a finite A far below does: the gradients are that one's, also at
    tokens whose step is 0."""
    B, T, D = 2, 70, 36
    g = torch.Generator().manual_seed(N)
    rn = lambda *s: torch.randn(*s, generator=g).to(dev)  # noqa: E731
    u, delta, Bm, C, z, dy = rn(B, T, D), rn(B, T, D), rn(B, T, N), rn(B, T, N), rn(B, T, D), rn(B, T, D)
    A, s0, ds = -torch.exp(rn(D, N)), rn(B, D, N), rn(B, D, N)
    if soft:
        delta[:, 5] = delta[:, 64] = float("-inf")
    else:
        delta = delta.abs() + 0.01
    far = A.clone()
    A[3, 1], A[7], A[35, 0] = (float("-inf"),) * 3
    far[3, 1], far[7], far[35, 0] = (-1e30,) * 3
    leaves = [t.requires_grad_() for t in (u, delta, A, Bm, C, z, s0)]
    y, fin = ssm_scan(*leaves[:5], z=z, delta_softplus=soft, initial_state=s0)
    got = torch.autograd.grad((y, fin), leaves, (dy, ds))
    form = (u, delta, far, Bm, C, None, z, None, soft, s0, dy, ds)
    ref, env = (R.scan_grads(*form, absolute=a) for a in (False, True))
    for x, i, name in zip(got, (0, 1, 2, 3, 4, 6, 8), ("u", "delta", "A", "B", "C", "z", "initial_state")):
        R.near(x, ref[i], 24 * (T + 16) * R.U * env[i], F32, name)


# ---- forward-mode derivatives ---------------------------------------------------------------------------
def test_forward_mode_is_refused(dev):
    """A dual tensor does not require a gradient and has storage to read; its tangent would be dropped."""
    fw = torch.autograd.forward_ad
    rn = lambda *s: torch.randn(*s, device=dev)  # noqa: E731
    u, A, Bm, w, state, pool = rn(1, 8, 8), -rn(8, 4).exp(), rn(1, 8, 4), rn(8, 4), rn(1, 3, 8), rn(1, 8, 4)
    cu, slots = torch.tensor([0, 8], dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    calls = [
        lambda d: ssm_scan(d(u), u, A, Bm, Bm), lambda d: ssm_scan(u, u, d(A), Bm, Bm),
        lambda d: ssm_scan(u, u, A, Bm, Bm, initial_state=d(pool)), lambda d: ssm_scan(u, u, A, Bm, Bm, z=d(u)),
        lambda d: ssm_scan_varlen(u, d(u), A, Bm, Bm, cu), lambda d: ssm_decode_step(u[:, 0], u[:, 0], A, Bm[:, 0],
                                                                                    Bm[:, 0], d(pool)),
        lambda d: short_conv(d(u), w), lambda d: short_conv(u, d(w)),
        lambda d: short_conv(u, w, initial_state=d(state)),
        lambda d: short_conv_varlen(u, d(w), cu), lambda d: short_conv_decode_step(d(u[:, 0]), w, state),
        lambda d: layer_norm(d(u)), lambda d: layer_norm(u, d(w[:, 0].contiguous())),
    ]
    with fw.dual_level():
        for call in calls:
            call(lambda t: t)  # tensors without a tangent are taken there too
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="forward-mode"):
                    call(lambda t: fw.make_dual(t, torch.ones_like(t)))


# ---- calls without tokens at the C entries ------------------------------------------------------------------
def test_no_tokens_leave_the_initial_state(dev):
    """T = 0 with sequences: the final state is the initial one, zeros without one, as in the packed calls; given as
    one buffer it stays."""
    lib, stream = L.lib(), torch.cuda.current_stream(dev).cuda_stream
    p = lambda t: ctypes.c_void_p(None if t is None else t.data_ptr())  # noqa: E731
    x = torch.zeros(64, device=dev)
    st = (ctypes.c_int64 * 14)(*([64] * 14))
    s0 = torch.randn(3, 10, 5, device=dev)

    def scan(a, b):
        return lib.triune_hip_ssm_scan(p(x), p(x), None, p(x), p(x), p(x), None, None, 0, st, 1, p(a), p(x), p(b), None,
                                       3, 0, 10, 1, 5, 0, None, 0, stream)

    for a in (s0, None):
        b = torch.full_like(s0, 7.0)
        assert scan(a, b) == 0
        assert torch.equal(b, torch.zeros_like(s0) if a is None else s0)
    keep = s0.clone()
    assert scan(s0, s0) == 0 and scan(s0, None) == 0 and torch.equal(s0, keep)
    for code, dtype in ((0, F32), (1, BF), (2, torch.float16)):
        c0 = torch.randn(3, 3, 11, device=dev).to(dtype)
        w = torch.zeros(44, device=dev)
        for a in (c0, None):
            b = torch.full_like(c0, 7.0)
            assert lib.triune_hip_short_conv(p(x), p(w), None, code, 0, st, 1, p(a), p(b), p(x), 3, 0, 11, 4,
                                             stream) == 0
            assert torch.equal(b, torch.zeros_like(c0) if a is None else c0)


# ---- output buffers and slots -------------------------------------------------------------------------------
def test_out_rows_of_two_dims_that_overlap_are_refused(dev):
    """Strides that each span a row but put rows of several sequences on one another; interleaved rows are taken."""
    u = torch.randn(2, 8, 8, device=dev)
    A, Bm, w = -torch.ones(8, 4, device=dev), torch.randn(2, 8, 4, device=dev), torch.randn(8, 4, device=dev)
    flat = torch.zeros(256, device=dev)
    for st in ((8, 8, 1), (16, 8, 1), (56, 8, 1), (8, 12, 1)):
        out = flat.as_strided((2, 8, 8), st)
        with pytest.raises(ValueError, match="overlap"):
            ssm_scan(u, u, A, Bm, Bm, out=out)
        with pytest.raises(ValueError, match="overlap"):
            short_conv(u, w, out=out)
    for st in ((64, 8, 1), (8, 16, 1), (9, 18, 1), (100, 10, 1)):
        out = flat.as_strided((2, 8, 8), st)
        assert torch.equal(ssm_scan(u, u, A, Bm, Bm, out=out)[0], ssm_scan(u, u, A, Bm, Bm)[0])
        assert torch.equal(short_conv(u, w, out=out)[0], short_conv(u, w)[0])


def test_wide_slots_are_outside_the_pool(dev):
    """int64 slots past 32 bits are outside the pool, not the row that their low half names; slots are integers."""
    D, N = 8, 4
    u, Bm, w = torch.randn(3, D, device=dev), torch.randn(3, N, device=dev), torch.randn(D, 4, device=dev)
    A = -torch.ones(D, N, device=dev)
    pool, cpool = torch.randn(4, D, N, device=dev), torch.randn(4, 3, D, device=dev)
    slots = torch.tensor([2, (1 << 32) + 1, -(1 << 32)], device=dev)
    cu = torch.tensor([0, 1, 2, 3], device=dev, dtype=torch.int32)
    near = torch.tensor([2, 4, -1], device=dev, dtype=torch.int32)  # the same rows, the others just outside
    for call, s in (
            (lambda s, k: ssm_decode_step(u, u, A, Bm, Bm, s, inplace=True, slots=k), pool),
            (lambda s, k: ssm_scan_varlen(u, u, A, Bm, Bm, cu, state_pool=s, slots=k), pool),
            (lambda s, k: short_conv_decode_step(u, w, s, inplace=True, slots=k), cpool),
            (lambda s, k: short_conv_varlen(u, w, cu, state_pool=s, slots=k), cpool)):
        a, b = s.clone(), s.clone()
        ya, yb = call(a, slots)[0], call(b, near)[0]
        assert torch.equal(a, b) and torch.equal(ya, yb) and torch.equal(a[[0, 1, 3]], s[[0, 1, 3]])
        for bad in (near.float(), near >= 0):
            with pytest.raises(TypeError, match="slots"):
                call(s.clone(), bad)


# ---- packed prompts, one far longer than the rest -----------------------------------------------------------
@pytest.mark.parametrize("place", [0, 30, 65])
@torch.no_grad()
def test_one_long_prompt_among_many_short_ones(dev, place):
    """Sequences enough to fill the chip, of which two are cut: states in a pool, one row padded, lengths on both
    sides of the longest that stays whole (512) and of a segment (128), empty ones."""
    lens = [ln for ln in (0, 1, 40, 128, 129, 512, 513, 33) for _ in range(2)] + [7, 19, 0, 64, 31] * 10
    lens[place:place] = [5001]
    n, D, N, total = len(lens), 1000, 16, sum(lens)
    assert S.plan_on(torch.zeros(1, device=dev), "triune_hip_ssm_scan_varlen_workspace_size", n, total, D, 1, N, 0) > 0
    g = torch.Generator().manual_seed(place)
    rn = lambda *s: torch.randn(*s, generator=g).to(dev)  # noqa: E731
    u, delta, Bm, C, z = rn(total, D), rn(total, D) - 4, rn(total, N), rn(total, N), rn(total, D)
    A, Dp, pool = -torch.exp(rn(D, N)), rn(D), rn(n + 2, D, N)
    before, slots = pool.clone(), torch.randperm(n + 2, generator=g)[:n].to(torch.int32)
    pad = lens.index(129)
    slots[pad] = -1
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    y, _ = ssm_scan_varlen(u, delta, A, Bm, C, cu.to(dev), Dp, z, state_pool=pool, slots=slots.to(dev))
    near = [i for i, ln in enumerate(lens) if ln > 100] + [i for i, ln in enumerate(lens) if ln <= 40][::7]
    for i in near:
        c, sl = slice(int(cu[i]), int(cu[i + 1])), int(slots[i])
        s0 = None if sl < 0 else before[sl:sl + 1]
        part = [t[None, c] for t in (u, delta)] + [A] + [t[None, c] for t in (Bm, C)]
        ry, rs, ey, es, _ = R.scan(*part, Dp, z[None, c], s0=s0)
        R.near(y[None, c], ry, ey, F32, f"sequence {i} of {lens[i]}")
        if sl >= 0:
            R.near(pool[sl:sl + 1], rs, es, F32, f"state {i} of {lens[i]}")
    rest = [r for r in range(n + 2) if r not in slots.tolist()]
    assert torch.equal(pool[rest], before[rest])
    again = before.clone()
    y2, _ = ssm_scan_varlen(u, delta, A, Bm, C, cu.to(dev), Dp, z, state_pool=again, slots=slots.to(dev))
    assert torch.equal(y, y2) and torch.equal(pool, again)


# ---- one token's terms at a time ----------------------------------------------------------------------------
@pytest.mark.parametrize("units", [0, 1])
def test_gradients_of_single_tokens_of_a_long_prompt(dev, units):
    """Upstream at one token and input at one: dC, dB, dA and the rest hold that pair's terms alone, with the roundings
    of the tokens between, so a term that a tile or segment drops or takes twice shows, which a bound on the sum over
    thousands of tokens would let pass."""
    T, D, N = 4430, 12, 5
    g = torch.Generator().manual_seed(1)
    rn = lambda *s: torch.randn(*s, generator=g).to(dev)  # noqa: E731
    for src, dst in ((0, 0), (0, 31), (31, 32), (2047, 2049), (2015, 2080), (4416, 4429), (4429, 4429)):
        u, dy = torch.zeros(1, T, D, device=dev), torch.zeros(1, T, D, device=dev)
        u[:, src], dy[:, dst] = rn(1, D), rn(1, D)
        delta, A, Bm, C, Dp = rn(1, T, D) - 5, -torch.exp(rn(D, N)), rn(1, T, N), rn(1, T, N), rn(D)
        _, _, kept = S._scan(u, delta, A, Bm, C, Dp, None, None, True, None, None, True, units << 8)
        got = S._scan_bwd(u, delta, A, Bm, C, Dp, None, None, True, kept, dy, None, False, units << 8)
        form = (u, delta, A, Bm, C, Dp, None, None, True, None, dy, None)
        ref, env = (R.scan_grads(*form, absolute=a) for a in (False, True))
        for name, x, r, e in zip("u delta A B C D".split(), got, ref, env):
            R.near(x, r, 24 * (dst - src + 33 + 16) * R.U * e, F32, f"{name} {src} {dst}")


# ---- the public training path in a graph --------------------------------------------------------------------
def test_training_steps_replay_from_a_graph(dev):
    """Forward and backward of each operator through its public call, captured together and replayed with new inputs
    and eager steps (on leaves of their own) between."""
    rn = lambda *s: torch.randn(*s, device=dev)  # noqa: E731
    B, T, D, N = 2, 200, 70, 16
    ops = [
        (lambda x, w, b: (layer_norm(x, w, b),), [rn(B * T, D).to(BF), rn(D).to(BF), rn(D).to(BF)]),
        (lambda x, w, b, s: short_conv(x, w, b, s), [rn(B, T, D).to(BF), rn(D, 4), rn(D), rn(B, 3, D).to(BF)]),
        (lambda u, d, A, Bm, C, Dp, z, bias, s: ssm_scan(u, d, A, Bm, C, Dp, z, bias, initial_state=s),
         [rn(B, T, D), rn(B, T, D), -rn(D, N).exp(), rn(B, T, N), rn(B, T, N), rn(D), rn(B, T, D), rn(D), rn(B, D, N)]),
    ]
    for op, data in ops:
        with torch.no_grad():
            ups = [torch.randn_like(t) for t in op(*data)]

        def step(inputs, ups=ups, op=op):
            leaves = [t.detach().requires_grad_() for t in inputs]
            return torch.autograd.grad(op(*leaves), leaves, ups)

        side = torch.cuda.Stream(device=dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            step(data)
        torch.cuda.current_stream(dev).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(data)
        for n in range(3):
            data[0].copy_(torch.randn(data[0].shape, generator=torch.Generator().manual_seed(n)))
            for t in out:
                t.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, step(data)):
                assert torch.equal(a, b)
        del graph


@torch.no_grad()
def test_thousands_of_packed_sequences(dev):
    """4200 sequences of two tokens, 64 states: the bits of the dense call."""
    n, D, N = 4200, 1088, 64
    g = torch.Generator().manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=g).to(dev)  # noqa: E731
    u, Bm, C, A, Dp = rn(n, 2, D), rn(n, 2, N), rn(n, 2, N), -rn(D, N).exp(), rn(D)
    cu = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device=dev)
    assert S.plan_on(u, "triune_hip_ssm_scan_varlen_workspace_size", n, 2 * n, D, 1, N, 0) > 0
    y, s = ssm_scan_varlen(u.flatten(0, 1), u.flatten(0, 1), A, Bm.flatten(0, 1), C.flatten(0, 1), cu, Dp)
    yd, sd = ssm_scan(u, u, A, Bm, C, Dp)
    assert torch.equal(y.view_as(yd), yd) and torch.equal(s, sd)
