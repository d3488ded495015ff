"""CPU: the sizes at which the decay attention entry points stop: what a grid holds, not what the states add up to.  Every
call ends at a check of its workspace or before it; none is launched."""

import pytest
from test_decay_host import BWD, DENSE, ENTRIES, VARLEN, base
from test_ssm_host import SHAPE, WORKSPACE, caller

import triune_amd._lib as L


@pytest.mark.parametrize("name,order", ENTRIES[:3])
def test_states_past_31_bits_are_taken(name, order):
    """4096 sequences of 64 heads of 128 x 128: 2^32 values of states."""
    flags = 2 << 8  # segments of 64 tokens, so that every call needs a workspace
    many = dict(B=4096, n=4096, rows=4096, H=64, Hk=64, Dk=128, Dv=128, T=128, total=4096 * 128, flags=flags)
    lib = L.lib()
    need = {"triune_hip_decay_attn": lambda: lib.triune_hip_decay_attn_workspace_size(4096, 128, 64, 64, 128, 128, flags),
            "triune_hip_decay_attn_varlen":
                lambda: lib.triune_hip_decay_attn_varlen_workspace_size(4096, 4096 * 128, 64, 64, 128, 128, flags),
            "triune_hip_decay_attn_bwd":
                lambda: lib.triune_hip_decay_attn_bwd_workspace_size(4096, 128, 64, 64, 128, 128, 1, 0, flags)}[name]()
    assert need >= 2 * 4 << 32  # two segments a sequence
    assert caller(name, order, **base(order))(**many) == WORKSPACE


def test_the_widest_heads_are_taken():
    lib = L.lib()
    wide = dict(B=1, H=65535, Hk=1, Dk=128, Dv=16384, T=1)
    assert lib.triune_hip_decay_attn_bwd_workspace_size(1, 1, 65535, 1, 128, 16384, 0, 0, 0) >= 2 * 4 * 65535 * 128 * 16384
    assert caller("triune_hip_decay_attn_bwd", BWD, **base(BWD))(**wide) == WORKSPACE


def test_gradients_past_32_bits_of_q_are_taken():
    """2^22 tokens of 16 heads of 128 key dims, 2^33 values; shared heads add theirs up in a loop."""
    size = L.lib().triune_hip_decay_attn_bwd_workspace_size
    assert size(64, 1 << 16, 16, 16, 128, 32, 1, 0, 0) > 0
    assert size(64, 1 << 16, 16, 4, 128, 32, 1, 0, 0) > 2 * 4 << 33
    assert size(1 << 15, 1 << 16, 16, 16, 128, 32, 1, 0, 0) == 0  # 2^29 chunks


def test_grids_are_refused():
    """2^16 sequences of 64 heads of 128 x 128: a join of 2^26 workgroups, where there is one; 2^24 work items."""
    dense = caller("triune_hip_decay_attn", DENSE, **base(DENSE))
    varlen = caller("triune_hip_decay_attn_varlen", VARLEN, **base(VARLEN))
    join = dict(B=1 << 16, n=1 << 16, rows=1 << 16, H=64, Hk=64, Dk=128, Dv=128, T=128, total=1 << 23, flags=2 << 8)
    assert dense(**join) == SHAPE and varlen(**join) == SHAPE
    items = dict(B=1 << 18, n=1 << 18, rows=1 << 18, H=64, Hk=64, Dk=128, Dv=128, T=64, total=1 << 18)
    assert dense(**items) == SHAPE and varlen(**items) == SHAPE
