"""GPU: fp32 and fp16 decay attention to bounds that its operands' own bits allow.  These types go through the fp32 matrix
cores, so the 260 units that bf16's derived operands may lose (decay_ref.py) are not theirs.

Units of U = 2^-24 at the ends, beside those of the decays:
  - any sizes: sums over the head dims, the chunk and the slices, Dk + Dv + 80
  - one to three tokens of one or two dims, whose other terms are zeros and add nothing: a sum of n products takes at most
    2 n (additions may cut), over the key dims, the value dims and the tokens, and sixteen more for the scale (twice), the
    sums of a gradient's parts, of a gate's four terms and of shared heads: 2 (Dk + Dv + T) + 16
An operand cut to two parts of bf16 is off by up to 128 units; test_decay_bits.py shows that the second bound sees that."""

import pytest
import torch
import decay_ref as D
from test_gpu_decay_attn import F32, HF, NAMES, inputs, train

pytestmark = pytest.mark.gpu


def check(args, s0, scale, units, flags=0):
    got, up = train(args, s0, scale, flags)
    ref = D.batch(*args, scale, s0, *up)
    bound = D.batch(*args, scale, s0, *up, bound=units)
    types = [args[0].dtype, F32, *(3 * [args[0].dtype]), args[3].dtype, F32]
    for n, a, r, b, t in zip(NAMES, got, ref, bound, types):
        D.near(a, r, D.U * b, t, n)


@pytest.mark.parametrize("dtype", [F32, HF])
@pytest.mark.parametrize("shape", [(2, 1, 4, 2, 64, 64), (1, 33, 3, 3, 33, 65), (2, 100, 6, 2, 48, 80), (1, 130, 2, 2, 128, 128),
                                   (2, 200, 4, 4, 16, 8)])
@pytest.mark.parametrize("flags", [0, 2 << 8])
def test_any_sizes(dev, shape, dtype, flags):
    *args, s0 = inputs(dev, *shape, dtype)
    _, T, H, Hk, Dk, Dv = shape
    check(args, s0, 0.3, Dk + Dv + 80 + (64 if H > Hk else 0), flags)


@pytest.mark.parametrize("dtype", [F32, HF])
@pytest.mark.parametrize("T,Dk,Dv", [(1, 1, 1), (2, 1, 2), (3, 2, 1)])
def test_few_terms(dev, dtype, T, Dk, Dv):
    *args, s0 = inputs(dev, 4, T, 64, 64, Dk, Dv, dtype)
    check(args, s0, 0.3, 2 * (Dk + Dv + T) + 16)
