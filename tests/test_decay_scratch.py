"""CPU: gradients that are given what the forward left take no place for it in their own workspace."""

import ctypes

from test_decay_host import BWD, base
from test_ssm_host import FAKE, LAYOUT, WORKSPACE, caller

import triune_amd._lib as L


def test_scratch_without_what_the_forward_keeps():
    lib, flags, sizes = L.lib(), 2 << 8, (2, 640, 4, 2, 64, 64)  # segments of 64 tokens, shared heads
    call = caller("triune_hip_decay_attn_bwd", BWD, **base(BWD, T=640, flags=flags))
    kept = lib.triune_hip_decay_attn_workspace_size(*sizes, flags)
    need = lib.triune_hip_decay_attn_bwd_workspace_size(*sizes, 1, 0, flags)
    assert kept > 0 and need > 2 * kept
    odd = ctypes.c_void_p(0x1004)  # a size that is enough is followed by a check of the alignment; nothing is launched
    for own, kw in ((need, {}), (need - kept, {"fws": FAKE, "fwsb": kept})):
        assert call(ws=FAKE, wsb=own - 1, **kw) == WORKSPACE
        assert call(ws=odd, wsb=own, **kw) == LAYOUT
