"""Whether strided tensors share memory, as the clip and the update ask it before they write, against lists of addresses (no GPU)."""
import random

import pytest
import torch

from oregon_gpt_oss_patching_b200 import _binding, build


@pytest.fixture(scope="module")
def binding():
    build.build()
    return _binding.load()


def _addresses(t):
    """The addresses of all bytes of a tensor, with repetitions."""
    at = torch.zeros(t.shape, dtype=torch.int64)
    for d, (n, s) in enumerate(zip(t.shape, t.stride())):
        at += (torch.arange(n) * s).view([n if i == d else 1 for i in range(t.dim())])
    return [t.data_ptr() + t.element_size() * a + b for a in at.flatten().tolist() for b in range(t.element_size())]


def _distinct(t):
    return t.as_strided([n if s else 1 for n, s in zip(t.shape, t.stride())], t.stride(), t.storage_offset())


def _random_view(rng, flat):
    dims = rng.randint(1, 4)
    shape = [rng.choice([1, 2, 3, 5]) for _ in range(dims)]
    stride = [rng.choice([0, 1, 2, 3, 4, 6, 7, 12, 24, 35]) for _ in range(dims)]
    size = sum((n - 1) * s for n, s in zip(shape, stride)) + 1
    return flat.as_strided(shape, stride, rng.randint(0, min(30, flat.numel() - size)))


def test_against_addresses(binding):
    rng = random.Random(1)
    both = {True: 0, False: 0}
    for _ in range(4000):
        flat = torch.zeros(600)
        # two types in one buffer: 2 bytes against 4
        other = rng.choice([flat, flat.view(torch.bfloat16)[:600]])
        a, b = _random_view(rng, flat), _random_view(rng, other)
        shared = bool(set(_addresses(a)) & set(_addresses(b)))
        assert binding.share_memory(a, b) == binding.share_memory(b, a) == shared, (a.shape, a.stride(), b.shape, b.stride())
        mine = _addresses(_distinct(a))
        assert binding.shares_with_itself(a) == (len(set(mine)) < len(mine)), (a.shape, a.stride())
        both[shared] += 1
    assert min(both.values()) > 500


def test_slices_and_permutations_of_one_buffer(binding):
    rng = random.Random(2)
    for _ in range(500):
        base = torch.zeros([rng.randint(1, 6) for _ in range(4)])

        def view():
            v = base
            for d in range(4):
                lo = rng.randrange(v.shape[d])
                v = v[(slice(None),) * d + (slice(lo, rng.randint(lo + 1, v.shape[d]), rng.randint(1, 3)),)]
            return v.permute(rng.sample(range(4), 4))

        a, b = view(), view()
        assert binding.share_memory(a, b) == bool(set(_addresses(a)) & set(_addresses(b)))
        assert not binding.shares_with_itself(a)


def test_large_tensors_are_told_apart_at_once(binding):
    big = torch.zeros(1, dtype=torch.bfloat16).as_strided((4096, 100_000), (0, 0))
    wide = torch.empty(4096 * 4096, dtype=torch.bfloat16).view(4096, 4096)
    assert not binding.share_memory(wide[:, :2048], wide[:, 2048:]) and not binding.share_memory(wide[:, ::2].t(), wide[:, 1::2])
    assert binding.share_memory(wide[:, :2049], wide[:, 2048:].t()) and binding.share_memory(wide, wide.t())
    assert not binding.share_memory(big, wide) and not binding.shares_with_itself(wide.t()) and not binding.shares_with_itself(big)
    empty = wide[:0]
    assert not binding.share_memory(empty, wide) and not binding.share_memory(wide, empty) and not binding.shares_with_itself(empty)
