"""GPU: decay attention against its 64-bit closed form: dense, packed and single-token calls, gradients, odd sizes, strides,
steep and infinite gates, segments, refusals."""

import pytest
import torch
import decay_ref as D

import triune_amd.decay as M
from triune_amd import decay_attn, decay_attn_decode_step, decay_attn_varlen

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
NAMES = "o final dq dk dv dg ds0".split()


def inputs(dev, B, T, H, Hk, Dk, Dv, dtype=F32, gdt=F32, head=False, steep=0.2, seed=0):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    gate = -steep * (rn(H) if head else rn(B, T, H)).abs()
    x = [t.to(dtype).to(dev) for t in (rn(B, T, Hk, Dk), rn(B, T, Hk, Dk), rn(B, T, H, Dv))]
    return (*x, gate.to(gdt).to(dev), rn(B, H, Dk, Dv).to(dev))


def ups(o, fin, seed=9):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(o.shape, generator=g).to(o.dtype).to(o.device),
            torch.randn(fin.shape, generator=g).to(fin.device))


def check(got, args, scale=1.0, s0=None, up=(None, None), what=""):
    q, k, v, g = args
    T, head = v.shape[1], g.dim() == 1
    ref = D.batch(q, k, v, g, scale, s0, *up)
    e = D.ends(q.shape[-1], v.shape[-1], v.shape[0] * T if head else 0, head or v.shape[2] != q.shape[2])
    bound = D.batch(q, k, v, g, scale, s0, *up, bound=e)
    types = [q.dtype, F32, q.dtype, q.dtype, q.dtype, g.dtype, F32]
    for n, a, r, b, t in zip(NAMES, got, ref, bound, types):
        if a is not None:
            D.near(a, r, D.U * b, t, f"{what} {n}")


def train(args, s0, scale=1.0, flags=0, seed=9):
    """All outputs and gradients, and what came in from above; flags force a segment's length."""
    q, k, v, g = args
    o, fin, kept = M._attn(q, k, v, g, scale, s0, None, flags)
    up = ups(o, fin, seed)
    grads = M._attn_bwd(q, k, v, g, scale, s0, *up, True, flags, kept)
    if kept is not None:  # the same without what the forward left
        again = M._attn_bwd(q, k, v, g, scale, s0, *up, True, flags)
        assert all(torch.equal(a, b) for a, b in zip(grads, again))
    return (o, fin, *grads), up


# B, T, H, Hk, Dk, Dv
SHAPES = [(1, 1, 1, 1, 1, 1), (2, 1, 4, 2, 64, 64), (1, 31, 2, 1, 16, 8), (2, 32, 2, 2, 32, 32), (1, 33, 3, 3, 33, 65),
          (2, 63, 2, 1, 64, 17), (1, 64, 4, 4, 128, 64), (1, 65, 2, 2, 65, 128), (2, 100, 6, 2, 48, 80),
          (1, 130, 2, 2, 128, 128), (1, 70, 3, 1, 100, 200), (1, 97, 2, 2, 7, 130), (1, 200, 2, 2, 64, 64)]


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("shape", SHAPES)
def test_outputs_and_gradients(dev, shape, dtype):
    *args, s0 = inputs(dev, *shape, dtype)
    got, up = train(args, s0, 0.3)
    check(got, args, 0.3, s0, up)


@pytest.mark.parametrize("dtype", [F32, BF, HF])
def test_constant_and_16_bit_gates(dev, dtype):
    *args, s0 = inputs(dev, 2, 150, 6, 3, 40, 72, dtype, head=True)
    got, up = train(args, s0)
    check(got, args, 1.0, s0, up, "constant")
    *args, s0 = inputs(dev, 2, 90, 4, 4, 64, 64, dtype, gdt=dtype)
    got, up = train(args, s0, -0.5)
    check(got, args, -0.5, s0, up, "gates in the io dtype")


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("flags", [2 << 8, 4 << 8])
@pytest.mark.parametrize("T", [65, 128, 129, 200, 257, 330])
def test_segments(dev, dtype, flags, T):
    """Two to six segments: what the walks form and the join carries, forwards and backwards."""
    *args, s0 = inputs(dev, 2, T, 4, 2, 64, 48, dtype, steep=0.02)
    got, up = train(args, s0, 0.125, flags)
    check(got, args, 0.125, s0, up)


def test_without_states(dev):
    *args, _ = inputs(dev, 1, 80, 2, 2, 32, 32)
    o, fin = decay_attn(*args)
    check((o, fin), args)
    leaves = [x.detach().requires_grad_() for x in args]
    o, fin = decay_attn(*leaves)
    up = ups(o, fin)
    for pick in ((0,), (1,)):  # one output's gradient alone
        grads = torch.autograd.grad([(o, fin)[i] for i in pick], leaves, [up[i] for i in pick], retain_graph=True)
        have = tuple(u if i in pick else torch.zeros_like(u) for i, u in enumerate(up))
        check((o, fin, *grads), args, 1.0, None, have)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_steep_and_resetting_gates(dev, dtype):
    """Gates of hundreds and -inf between ones near 0: decays behind them keep their own precision, and the gates'
    gradients, of pairs that span a token only, theirs."""
    *args, s0 = inputs(dev, 2, 140, 3, 3, 32, 32, dtype, steep=1e-3)
    for t, x in ((5, -200.0), (31, float("-inf")), (32, -90.0), (70, -1e30), (71, float("-inf")), (139, -30.0)):
        args[3][:, t, 1] = x
    args[3][:, ::3, 2] = -7.0
    got, up = train(args, s0)
    assert all(bool(x.isfinite().all()) for x in got)
    check(got, args, 1.0, s0, up)
    for flags in (2 << 8,):
        got, up = train(args, s0, 1.0, flags)
        check(got, args, 1.0, s0, up)


def test_gates_above_zero_count_as_zero(dev):
    *args, s0 = inputs(dev, 1, 50, 2, 2, 16, 16)
    args[3][0, 3::7] = 5.0
    args[3][0, 20, 1] = 0.0
    got, up = train(args, s0)
    check(got, args, 1.0, s0, up)
    assert bool((got[5][0, 3::7] == 0).all()) and float(got[5][0, 20, 1]) != 0
    args[3] = torch.tensor([-0.1, 0.5], device=dev)
    got, up = train(args, s0)
    check(got, args, 1.0, s0, up)
    assert float(got[5][1]) == 0


@pytest.mark.parametrize("dtype", [F32, BF, HF])
def test_not_finite_values_stay_in_their_sequence_and_head(dev, dtype):
    *args, s0 = inputs(dev, 3, 70, 4, 2, 32, 32, dtype)
    want, up = train(args, s0)
    bad = [x.clone() for x in args]
    bad[2][1, 40, 3, 5] = float("nan")
    bad[3][2, 10, 0] = float("nan")
    got, _ = train(bad, s0)
    assert bool(got[0][1, 40:, 3, 5].isnan().all()) and bool(got[0][2, 10:, 0].isnan().all())
    for a, b in zip(got[:2], want[:2]):
        assert torch.equal(a[0], b[0])
    assert torch.equal(got[0][1, :, :3], want[0][1, :, :3]) and torch.equal(got[0][1, :32], want[0][1, :32])
    assert torch.equal(got[0][2, :, 1:], want[0][2, :, 1:])
    assert torch.equal(got[2][0], want[2][0]) and torch.equal(got[4][2, :, 1:], want[4][2, :, 1:])


@pytest.mark.parametrize("dtype", [F32, BF])
def test_layouts(dev, dtype):
    """Views of one projection, heads in front of tokens, steps between tokens, unaligned starts, innermost strides that are
    not 1, broadcast values and gates."""
    B, T, H, Dk, Dv = 2, 75, 3, 24, 40
    g = torch.Generator().manual_seed(3)
    flat = torch.randn(B, T, H * (2 * Dk + Dv) + 5, generator=g).to(dtype).to(dev)[..., 3:-2]
    q, k = (flat[..., i * H * Dk:(i + 1) * H * Dk].unflatten(-1, (H, Dk)) for i in range(2))
    v = flat[..., 2 * H * Dk:].unflatten(-1, (H, Dv))
    gate = -torch.rand(B, H, T, generator=g).to(dev).transpose(1, 2)
    s0 = torch.randn(B, H, Dv, Dk, generator=g).to(dev).transpose(2, 3)
    base = (q, k, v, gate)
    turned = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    wide = [torch.randn(B, 2 * T, H, x.shape[-1], generator=g).to(dtype).to(dev)[:, ::2] for x in (q, k, v)]
    inner = [x.transpose(-1, -2).contiguous().transpose(-1, -2) for x in (q, k, v)]
    shared = [x[:, :, :1].expand(-1, -1, H, -1) for x in (q, k, v)]
    once = [x[:1, :1].expand(B, T, -1, -1) for x in (q, k, v)]
    for what, args in (("views", base), ("turned", (*turned, gate)), ("steps", (*wide, gate)), ("inner", (*inner, gate)),
                       ("shared", (*shared, gate[:, :, :1].expand(-1, -1, H))), ("once", (*once, gate[:, :1].expand(-1, T, -1)))):
        leaves = [x.detach().requires_grad_() for x in (*args, s0)]
        o, fin = decay_attn(*leaves[:4], initial_state=leaves[4])
        up = ups(o, fin)
        check((o, fin, *torch.autograd.grad((o, fin), leaves, up)), args, 1.0, s0, up, what)
    want, _ = decay_attn(*base, initial_state=s0)
    buf = torch.full((B, H, T, Dv + 3), 7.0, device=dev, dtype=dtype)
    out = buf.transpose(1, 2)[..., 1:Dv + 1]
    got, _ = decay_attn(*base, initial_state=s0, out=out)
    assert got is out and torch.equal(out, want) and bool((buf[..., 0] == 7).all() and (buf[..., Dv + 1:] == 7).all())


def test_gradients_of_shared_heads_through_autograd(dev):
    """A gate that is broadcast over tokens by the caller, one used twice, and a leaf under several uses."""
    q, k, v, g, s0 = inputs(dev, 2, 40, 4, 1, 16, 24, head=True)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, g)]
    o, fin = decay_attn(leaves[0], leaves[0], leaves[2], leaves[3].expand(2, 40, 4))
    up = ups(o, fin)
    dq, dv, dg = torch.autograd.grad((o, fin), [leaves[0], leaves[2], leaves[3]], up)
    r = D.batch(q, q, v, g, 1.0, None, *up)
    b = D.batch(q, q, v, g, 1.0, None, *up, bound=D.ends(16, 24, 80, True))
    D.near(dq, r[2] + r[3], D.U * (b[2] + b[3]), F32, "dq + dk")
    D.near(dv, r[4], D.U * b[4])
    D.near(dg, r[5], D.U * b[5])


@pytest.mark.parametrize("dtype", [F32, BF, HF])
def test_gradients_against_differences(dev, dtype):
    """A step along each input by a power of two, in a direction of powers of two, so that both ends are numbers of the
    type; the outputs are linear in q, k and v and nearly so in g there."""
    *args, s0 = inputs(dev, 1, 96, 2, 1, 32, 32, dtype)
    leaves = [x.detach().requires_grad_() for x in (*args, s0)]
    o, fin = decay_attn(*leaves[:4], initial_state=leaves[4], scale=0.25)
    up = ups(o, fin)
    grads = torch.autograd.grad((o, fin), leaves, up)
    for i, grad in enumerate(grads):
        h = 2.0**-9 if i == 3 else 2.0**-2
        step = torch.sign(torch.randn(grad.shape, generator=torch.Generator().manual_seed(i))).to(dev) * h
        ends = []
        for s in (step, -step):
            x = [t.double() for t in (*args, s0)]
            x[i] = x[i] + s.double()
            r = D.batch(*x[:4], 0.25, x[4])
            ends.append(float((r[0] * D.d64(up[0])).sum() + (r[1] * D.d64(up[1])).sum()))
        want, got = (ends[0] - ends[1]) / 2, float((grad.double() * step.double()).sum())
        # each gradient is off by half a step of its type; a difference in g by h^2 / 6 of a third derivative, which a
        # decay over all 96 tokens has at 96 times the first
        tol = float((grad.double().abs() * step.double().abs()).sum()) * (torch.finfo(grad.dtype).eps + 2.0**-12)
        tol += 0 if i != 3 else (h * 96) ** 2 / 6 * float((grad.double() * step.double()).abs().sum())
        assert abs(got - want) <= tol, (i, got, want, tol)


# ---- packed -----------------------------------------------------------------------------------------------------
@torch.no_grad()
@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("lens", [[1], [5, 0, 64, 33, 1], [300, 7, 129], [0, 0, 3], [40] * 9, [1000, 1, 2]])
def test_packed(dev, dtype, lens):
    """Ragged sequences over pool slots, with rows in front of and behind them that stay as they were."""
    H, Hk, Dk, Dv, lead, n = 4, 2, 32, 40, 3, len(lens)
    total = sum(lens) + lead + 6
    q, k, v, g, _ = inputs(dev, 1, total, H, Hk, Dk, Dv, dtype)
    q, k, v, g = (x[0] for x in (q, k, v, g))
    v[:lead], g[-2:] = float("nan"), float("nan")
    cu = (torch.tensor([0, *lens]).cumsum(0) + lead).to(torch.int32).to(dev)
    pool = torch.randn(n + 2, H, Dk, Dv, generator=torch.Generator().manual_seed(1)).to(dev)
    before = pool.clone()
    slots = torch.tensor([(3 * i + 1) % (n + 2) if (n + 2) % 3 else (i + 1) % (n + 2) for i in range(n)], dtype=torch.int32)
    out = torch.full((total, H, Dv), 5.0, device=dev, dtype=dtype)
    o, got = decay_attn_varlen(q, k, v, g, cu, scale=0.2, out=out, state_pool=pool, slots=slots.to(dev))
    assert o is out and got is pool
    idle = sorted(set(range(n + 2)) - set(slots.tolist()))
    assert torch.equal(pool[idle], before[idle])
    assert bool((out[:lead] == 5).all()) and bool((out[lead + sum(lens):] == 5).all())
    o2, fin = decay_attn_varlen(q[None], k[None], v[None], g[None], cu, before[slots.long().to(dev)], 0.2)
    for i, m in enumerate(lens):
        a = int(cu[i])
        part, s0 = [x[None, a:a + m] for x in (q, k, v, g)], before[int(slots[i])][None]
        if m:
            check((out[None, a:a + m], pool[int(slots[i])][None]), part, 0.2, s0, what=f"sequence {i}")
            assert torch.equal(o2[0, a:a + m], out[a:a + m])
        else:
            assert torch.equal(pool[int(slots[i])], before[int(slots[i])])
        assert torch.equal(fin[i], pool[int(slots[i])])


@torch.no_grad()
def test_packed_padded_rows_and_bad_offsets(dev):
    """Slots outside the pool start from zero and keep nothing; offsets are cut to the packed rows."""
    q, k, v, g, _ = inputs(dev, 1, 90, 2, 2, 32, 32)
    q, k, v, g = (x[0] for x in (q, k, v, g))
    pool = torch.randn(3, 2, 32, 32, device=dev)
    before = pool.clone()
    cu = torch.tensor([0, 30, 60, 90], dtype=torch.int32, device=dev)
    o, _ = decay_attn_varlen(q, k, v, g, cu, state_pool=pool, slots=torch.tensor([-1, 2, 7], device=dev))
    assert torch.equal(pool[:2], before[:2])
    zero, fin = decay_attn_varlen(q, k, v, g, cu, initial_state=torch.stack([0 * pool[0], before[2], 0 * pool[0]]))
    assert torch.equal(o, zero) and torch.equal(fin[1], pool[2])
    wild = torch.tensor([-40, 30, 2_000_000_000], dtype=torch.int64, device=dev)
    o, fin = decay_attn_varlen(q, k, v, g, wild)
    want, fin2 = decay_attn_varlen(q, k, v, g, torch.tensor([0, 30, 90], dtype=torch.int32, device=dev))
    assert torch.equal(o, want) and torch.equal(fin, fin2)


@torch.no_grad()
@pytest.mark.parametrize("dtype", [F32, BF])
def test_long_packed_sequences_are_cut_in_place(dev, dtype):
    """Sequences long enough for segments, whose last one writes the pool row that the first one reads."""
    lens = [2000, 100, 3000, 1, 700]
    q, k, v, g, _ = inputs(dev, 1, sum(lens), 2, 2, 64, 64, dtype, steep=0.01)
    cu = torch.tensor([0, *lens]).cumsum(0).to(torch.int32).to(dev)
    pool = torch.randn(5, 2, 64, 64, device=dev)
    start = pool.clone()
    assert M.plan_on(q, "triune_hip_decay_attn_varlen_workspace_size", 5, sum(lens), 2, 2, 64, 64, 0) > 0
    o, _ = decay_attn_varlen(q, k, v, g, cu, state_pool=pool, slots=torch.arange(5, device=dev))
    for i in range(5):
        part = [x[:, int(cu[i]):int(cu[i + 1])] for x in (q, k, v, g)]
        check((o[:, int(cu[i]):int(cu[i + 1])], pool[i:i + 1]), part, 1.0, start[i:i + 1], what=f"sequence {i}")


# ---- single tokens ------------------------------------------------------------------------------------------------
@torch.no_grad()
@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (3, 4, 2, 64, 64), (5, 6, 6, 33, 65), (2, 2, 1, 128, 300), (4, 3, 3, 7, 5),
                                   (2, 2, 2, 128, 128), (70, 2, 2, 16, 32)])
def test_decode_step(dev, shape, dtype):
    B, H, Hk, Dk, Dv = shape
    q, k, v, g, s0 = inputs(dev, B, 1, H, Hk, Dk, Dv, dtype)
    o, s = decay_attn_decode_step(q, k, v, g, s0, scale=0.4)
    check((o, s), (q, k, v, g), 0.4, s0)
    pool = torch.randn(B + 4, H, Dk, Dv, generator=torch.Generator().manual_seed(2)).to(dev)
    before, slots = pool.clone(), (torch.arange(B) * 1 + 2).flip(0).to(torch.int32).to(dev)
    slots[0] = -1 if B > 1 else slots[0]
    o, s = decay_attn_decode_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], pool, 0.4, inplace=True, slots=slots)
    assert s is pool
    for b, r in enumerate(slots.tolist()):
        if r < 0:
            assert bool((o[b] == 0).all())
        else:
            check((o[b][None, None], pool[r][None]), [x[b:b + 1] for x in (q, k, v, g)], 0.4, before[r][None])
    idle = sorted(set(range(B + 4)) - set(slots.tolist()))
    assert torch.equal(pool[idle], before[idle])
    o2, s2 = decay_attn_decode_step(q, k, v, g, before, 0.4, slots=slots)
    assert torch.equal(o2[:, 0], o) and torch.equal(s2, pool)


@torch.no_grad()
@pytest.mark.parametrize("dtype", [F32, BF])
def test_prompts_and_steps_agree(dev, dtype):
    """A prompt in one call, and its start in one and the rest token by token, within the bounds of both."""
    *args, s0 = inputs(dev, 2, 50, 4, 2, 64, 32, dtype, head=True)
    o, fin = decay_attn(*(x[:, :41] for x in args[:3]), args[3], s0)
    outs = [o]
    for t in range(41, 50):
        o, fin = decay_attn_decode_step(*(x[:, t:t + 1] for x in args[:3]), args[3], fin, inplace=True)
        outs.append(o)
    check((torch.cat(outs, 1), fin), args, 1.0, s0)


# ---- other streams, devices' habits, refusals ------------------------------------------------------------------------
@torch.no_grad()
def test_two_streams_at_once(dev):
    """Calls with workspaces of their own on two streams at once give the bits of calls alone."""
    calls = [inputs(dev, 1, 3000, 2, 2, 64, 64, BF, seed=s) for s in range(2)]
    want = [decay_attn(*c[:4], initial_state=c[4]) for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=dev) for _ in calls]
    got = [[] for _ in calls]
    for _ in range(4):
        for c, s, r in zip(calls, streams, got):
            with torch.cuda.stream(s):
                r.append(decay_attn(*c[:4], initial_state=c[4]))
    torch.cuda.synchronize()
    for w, r in zip(want, got):
        for o, f in r:
            assert torch.equal(o, w[0]) and torch.equal(f, w[1])


def test_repeats_give_the_same_bits(dev):
    *args, s0 = inputs(dev, 2, 700, 6, 2, 64, 80, BF, head=True)
    first, _ = train(args, s0)
    for _ in range(3):
        again, _ = train(args, s0)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_empty_calls(dev):
    for B, T in ((0, 5), (2, 0)):
        *args, s0 = inputs(dev, B, T, 2, 2, 8, 8)
        leaves = [x.detach().requires_grad_() for x in (*args, s0)]
        o, fin = decay_attn(*leaves[:4], initial_state=leaves[4])
        assert o.shape == (B, T, 2, 8) and torch.equal(fin, s0)
        up = torch.randn_like(fin)
        grads = torch.autograd.grad((o, fin), leaves, (torch.zeros_like(o), up))
        assert torch.equal(grads[4], up) and all(not x.any() for x in grads[:4])
        with torch.no_grad():
            o, fin = decay_attn(*args, initial_state=s0)
            assert torch.equal(fin, s0) and fin.data_ptr() != s0.data_ptr() or B == 0
    q, k, v, g, s0 = inputs(dev, 1, 0, 2, 2, 8, 8)
    o, fin = decay_attn_varlen(q, k, v, g, torch.zeros(2, dtype=torch.int32), s0)
    assert torch.equal(fin, s0) and o.shape == v.shape
    o, s = decay_attn_decode_step(*(x[:0, :1] for x in inputs(dev, 1, 1, 2, 2, 8, 8)[:4]), s0[:0])
    assert o.shape == (0, 1, 2, 8) and s.shape[0] == 0


def test_refusals(dev):
    q, k, v, g, s0 = inputs(dev, 2, 8, 4, 2, 16, 16)
    bad = [
        (ValueError, "dim", lambda: decay_attn(q[0], k[0], v[0], g[0])),
        (ValueError, "q's shape", lambda: decay_attn(q, k[:, :7], v, g)),
        (ValueError, "leading dims", lambda: decay_attn(q, k, v[:1], g)),
        (ValueError, "divide", lambda: decay_attn(q, k, v[:, :, :3], g[:, :, :3])),
        (ValueError, "head dims", lambda: decay_attn(*(torch.zeros(1, 2, 1, 129, device=dev),) * 3, g[:1, :2, :1])),
        (ValueError, "g must be", lambda: decay_attn(q, k, v, g[:, :, :2])),
        (ValueError, "g must be", lambda: decay_attn(q, k, v, g[0])),
        (TypeError, "one dtype", lambda: decay_attn(q, k.half(), v, g)),
        (TypeError, "g must have", lambda: decay_attn(q, k, v, g.half())),
        (TypeError, "dtype", lambda: decay_attn(q.double(), k.double(), v.double(), g)),
        (ValueError, "initial_state", lambda: decay_attn(q, k, v, g, s0[:1])),
        (ValueError, "CPU|device", lambda: decay_attn(q, k, v, g.cpu())),
        (ValueError, "out must", lambda: decay_attn(q, k, v, g, out=torch.zeros_like(q))),
        (ValueError, "overlap", lambda: decay_attn(q, k, v, g, out=v[:1].expand_as(v))),
        (ValueError, "without gradients", lambda: decay_attn(q, k, v.clone().requires_grad_(), g, out=torch.empty_like(v))),
        (ValueError, "no gradient", lambda: decay_attn_varlen(q[0], k[0], v[0].clone().requires_grad_(), g[0],
                                                              torch.tensor([0, 8]))),
        (ValueError, "batch size 1", lambda: decay_attn_varlen(q, k, v, g, torch.tensor([0, 8]))),
        (ValueError, "needs slots", lambda: decay_attn_varlen(q[0], k[0], v[0], g[0], torch.tensor([0, 8]), state_pool=s0)),
        (ValueError, "state_pool must", lambda: decay_attn_varlen(q[0], k[0], v[0], g[0], torch.tensor([0, 8]),
                                                                  state_pool=s0.half(), slots=torch.tensor([0]))),
        (ValueError, "not both", lambda: decay_attn_varlen(q[0], k[0], v[0], g[0], torch.tensor([0, 8]), s0, state_pool=s0,
                                                           slots=torch.tensor([0]))),
        (ValueError, "one token", lambda: decay_attn_decode_step(q, k, v, g, s0)),
        (ValueError, "state has", lambda: decay_attn_decode_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], s0[:1])),
        (ValueError, "inplace", lambda: decay_attn_decode_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], s0.half(), inplace=True)),
        (TypeError, "slots", lambda: decay_attn_decode_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], s0,
                                                            slots=torch.zeros(2, device=dev))),
    ]
    for kind, match, call in bad:
        with pytest.raises(kind, match=match):
            call()
    fw = torch.autograd.forward_ad
    with fw.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        decay_attn(fw.make_dual(q, q), k, v, g)
    leaf = v.clone().requires_grad_()
    o, _ = decay_attn(q, k, leaf, g)
    dv, = torch.autograd.grad(o.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        dv.sum().backward()
