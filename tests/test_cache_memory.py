"""Which tensors count as sharing memory (no GPU needed), and caches that do so in part."""
import itertools

import pytest
import torch

from bkcore.attention import _share


def cells(t):
    """Addresses of a tensor's elements."""
    at = torch.zeros((), dtype=torch.int64)
    for n, s in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(n) * s
    return set((t.data_ptr() + at.flatten() * t.element_size()).tolist())


def test_sharing_is_exact_for_views_of_equal_strides():
    base = torch.zeros(4000)
    shapes = [(2, 3, 4, 5), (1, 2, 7, 3), (3, 1, 2, 2)]
    orders = list(itertools.permutations(range(4)))[::5]
    seen = set()
    for shape in shapes:
        for order in orders:
            for gap in (0, 2):
                stride, reach = [0] * 4, 1
                for i in order:                                   # innermost first, with gaps between
                    stride[i] = reach
                    reach = reach * shape[i] + gap
                for offset in list(range(0, 40)) + [60, 61, 119, 120, 150, 400]:
                    a, b = (torch.as_strided(base, shape, stride, o) for o in (7, 7 + offset))
                    want = bool(cells(a) & cells(b))
                    assert _share(a, b) == want and _share(b, a) == want, (shape, stride, offset)
                    seen.add(want)
    assert seen == {True, False}


def test_sharing_of_other_views():
    a = torch.zeros(2, 3, 4, 5)
    assert _share(a, a) and _share(a, a[:, :, 1:]) and _share(a, a.transpose(2, 3))
    assert not _share(a, torch.zeros(2, 3, 4, 5)) and not _share(a[:1], a[1:]) and not _share(a[:0], a)
    both = torch.zeros(2, 4, 2, 3, 5)                             # keys and values side by side in a slot
    k, v = both.permute(2, 0, 3, 1, 4)
    assert not _share(k, v)


def test_sharing_is_never_missed_between_views_of_any_strides():
    base = torch.zeros(3000)
    g = torch.Generator().manual_seed(0)
    r = lambda lo, hi: int(torch.randint(lo, hi, (), generator=g))
    seen = set()
    for _ in range(3000):
        a, b = (torch.as_strided(base, [r(1, 4) for _ in range(4)], [(0, 1, 2, 3, 5, 12, 60, 200)[r(0, 8)] for _ in range(4)], r(0, 300))
                for _ in range(2))
        share = bool(cells(a) & cells(b))
        seen.add(share)
        assert _share(a, b) or not share
        assert _share(a, b) == _share(b, a)
    assert seen == {True, False}


def test_prompts_and_caches_in_one_slab_a_sequence_do_not_share():
    slab = torch.zeros(3, 1000)                                   # prompt, keys, values of a sequence one behind the other
    k = slab[:, :160].view(3, 5, 2, 16).transpose(1, 2)
    kc, vc = (slab[:, at:at + 320].view(3, 2, 10, 16) for at in (160, 480))
    assert not _share(k, kc) and not _share(k, vc) and not _share(kc, vc)
    assert _share(k, slab[:, 159:479].view(3, 2, 10, 16)) and _share(vc, slab[:, 479:799].view(3, 2, 10, 16))


@pytest.mark.gpu
def test_caches_that_share_a_part_are_refused():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import bkcore
    rn = lambda *s: torch.randn(*s, device="cuda")
    long = rn(2, 2, 21, 16)
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    kept = long.clone()
    for a, b in ((long[:, :, :12], long[:, :, 1:13]), (long[:, :, 9:], long[:, :, :12]), (long[..., :12, :8], long[..., :12, 7:15])):
        D = a.shape[-1]
        with pytest.raises(ValueError, match="share"):
            bkcore.sliding_attention_step(rn(2, 4, D), rn(2, 2, D), rn(2, 2, D), a, b, pos, 8, 2)
        with pytest.raises(ValueError, match="share"):
            bkcore.sliding_cache_fill(rn(2, 2, 5, D), rn(2, 2, 5, D), a, b)
    for kv in ((long[:, :, 3:9], rn(2, 2, 6, 16)), (rn(2, 2, 6, 16), long[:, :, :6])):
        with pytest.raises(ValueError, match="share"):            # moving a cache's own content
            bkcore.sliding_cache_fill(*kv, long[:, :, :12], rn(2, 2, 12, 16))
    assert torch.equal(long, kept)
    new = rn(2, 2, 16)
    bkcore.sliding_attention_step(rn(2, 4, 16), new, new, long[:, :, :10], long[:, :, 10:20], pos, 8, 2)   # neighbours
    assert torch.equal(long[:, :, 0], new) and torch.equal(long[:, :, 10], new) and torch.equal(long[:, :, 1:10], kept[:, :, 1:10])
