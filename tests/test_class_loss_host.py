"""CPU checks of the class-score losses' C ABI: workspace sizes."""

import pytest

pytest.importorskip("torch")

from modern_fm_b200 import _lib  # noqa: E402


def test_policy_workspace_does_not_grow_with_the_tokens():
    """Its sums are those of one wave of blocks, however many tokens those walk."""
    f = _lib.lib().mfm_policy_workspace_bytes
    sizes = [f(1, n) for n in (0, 1, 100, 4096, 10**6, 2**31 - 1)]
    assert sizes == sorted(sizes) and 0 < sizes[0] and sizes[-1] <= 1 << 17
