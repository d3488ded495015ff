"""CPU: the segments that dense calls of decay attention are cut into, exactly."""

import pytest

import triune_amd._lib as L


def segments(B, T, H, flags=0):
    """Segments of a sequence of heads of 64, from the states and the sums that a workspace holds; 1: no workspace."""
    have = L.lib().triune_hip_decay_attn_workspace_size(B, T, H, H, 64, 64, flags)
    pad = lambda n: -(-n // 256) * 256  # noqa: E731
    sizes = {pad(4 * B * n * H * 64 * 64) + pad(8 * B * n * H): n for n in range(2, T // 64 + 2)}
    return 1 if have == 0 else sizes[have]


@pytest.mark.parametrize("T,n", [(1, 1), (64, 1), (65, 1), (127, 1), (128, 2), (191, 2), (192, 3), (640, 10)])
def test_automatic(T, n):
    assert segments(1, T, 1) == n


@pytest.mark.parametrize("units,n", [(1, 10), (2, 10), (3, 5), (4, 5), (5, 4), (6, 4), (20, 1), (255, 1)])
def test_forced_lengths_are_rounded_up_to_64_tokens(units, n):
    """640 tokens; flags force units of 32 tokens, which dense calls round up to whole chunks of the gradients."""
    assert segments(1, 640, 1, units << 8) == n


def test_lengths_of_one_segment_are_not_cut():
    """Of the lengths that test_gpu_decay_attn.py forces, 65 tokens by 64 or 128 and 128 by 128 are one segment or two."""
    assert [segments(2, T, 4, 2 << 8) for T in (65, 128, 129)] == [2, 2, 3]
    assert [segments(2, T, 4, 4 << 8) for T in (65, 128, 129)] == [1, 1, 2]
