"""The attention cache without a GPU: sizes at the end of their range."""
from __future__ import annotations

import pytest

import maivs_b200 as M

P = 4096  # an address that is aligned for every type; no call here gets as far as using it


def test_sizes_past_64_bits_are_refused():
    c = M.AttentionCache(3, 100, 2, 80, device=None)
    big = 2**64 + 4
    for kw in (dict(n_seqs=big), dict(capacity=big), dict(n_heads=big), dict(dim=big), dict(device=2**31), dict(device=2**32)):
        a = dict(n_seqs=1, capacity=8, n_heads=1, dim=64, device=None)
        a.update(kw)
        with pytest.raises(ValueError):
            M.AttentionCache(**a)
    with pytest.raises(ValueError):
        c.append(P, P, big, P, P)
    with pytest.raises(ValueError):
        c.append(P, P, 4, P, P, key_stride=2**64 + 160)
    with pytest.raises(ValueError):
        c.read(P, P, big, P, P)
    for kw in (dict(n_tokens=big), dict(n_query_heads=big), dict(max_rows=big), dict(max_tokens=big)):
        a = dict(n_tokens=4, n_query_heads=4)
        a.update(kw)
        with pytest.raises(ValueError):
            c.attend_workspace(**a)
    with pytest.raises(ValueError):
        c.attend(P, 4, 4, P, P, P, d_weights_in=P, d_weights_out=P, d_workspace=P, workspace_bytes=2**64 + 2**30)
    with pytest.raises(ValueError):
        c.attend_found_workspace(4, 4, big)
    with pytest.raises(ValueError):
        c.evict(P, big, P, P, 2 * P, d_workspace=P, workspace_bytes=2**30)
