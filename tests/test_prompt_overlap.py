"""Which views of one buffer share memory, as the prompt operators decide it, against
the elements that the views hold; CPU only."""

from __future__ import annotations

import random

import pytest
import torch

from local_kimi_amd.kernels.kda import _disjoint, _share


@pytest.mark.parametrize("seed", range(4))
def test_views_share_what_they_hold(seed):
    rng = random.Random(seed)
    base = torch.arange(400, dtype=torch.float32)

    def held(t):
        return set(t.flatten().tolist())

    seen = [0, 0]
    for _ in range(1000):
        shape = [rng.randint(1, 4) for _ in range(3)]
        strides = [rng.choice([0, 1, 2, 3, 4, 5, 7, 8, 12, 24, 48]) for _ in range(3)]
        a, b = (torch.as_strided(base, shape, strides, rng.randint(0, 60)) for _ in range(2))
        want = bool(held(a) & held(b))
        assert _share(a, b) == _share(b, a) == want, (shape, strides)
        seen[want] += 1
        # other strides: never taken for apart where they are not
        c = torch.as_strided(base, shape, [rng.choice([1, 2, 4, 16]) for _ in range(3)], rng.randint(0, 150))
        assert _share(a, c) or not held(a) & held(c)
    assert min(seen) > 100


def test_what_is_only_read_may_be_one_tensor():
    a, b, c = (torch.zeros(2, 3, 4) for _ in range(3))
    assert _disjoint([a, b], [c, c]) and _disjoint([a]) and not _disjoint([a, a])
    assert not _disjoint([a, b], [c, a]) and not _disjoint([a, b], [c, a[:, :, ::1]])
    wide = torch.zeros(2, 3, 8)
    assert _disjoint([wide[..., ::2], wide[..., 1::2]])
    assert not _disjoint([wide[..., :4], wide[..., 3:7]]) and not _disjoint([a], [c, a.flip(0).flip(0), a])
