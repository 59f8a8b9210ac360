"""_native.may_overlap: ranges apart, interleaved columns, and real overlaps (no GPU)."""
import itertools

import pytest
import torch


def test_told_apart_by_range_and_by_columns():
    from eraserdit_b200._native import may_overlap
    buf = torch.zeros(6, 100)
    assert not may_overlap(buf[:3], buf[3:])
    assert may_overlap(buf[:4], buf[3:])
    assert not may_overlap(buf[:, :40], buf[:, 40:])
    assert may_overlap(buf[:, :41], buf[:, 40:])
    assert not may_overlap(buf[:0], buf)
    assert not may_overlap(buf, torch.zeros(6, 100))
    # a column range that wraps around the period
    flat = buf.view(-1)
    late = flat.as_strided((5, 30), (100, 1), 85)  # columns 85..114 of each row
    assert not may_overlap(buf[:, 20:80], late)
    assert may_overlap(buf[:, 10:80], late)


def test_heads_of_a_projection_buffer():
    from eraserdit_b200._native import may_overlap
    buf = torch.zeros(2, 5, 12 * 64)
    heads = [buf[..., i * 64:(i + n) * 64].unflatten(-1, (n, 64)) for i, n in ((0, 4), (4, 2), (6, 6))]
    for a, b in itertools.combinations(heads, 2):
        assert not may_overlap(a, b) and not may_overlap(b, a)
    assert may_overlap(buf[..., :256].unflatten(-1, (4, 64)), buf[..., 192:320].unflatten(-1, (2, 64)))


def test_never_denies_an_overlap():
    """Against the elements' addresses, over many small views."""
    from eraserdit_b200._native import may_overlap
    buf = torch.zeros(64)
    views = [buf.as_strided(size, stride, off) for size in ((2, 3), (3, 2), (4, 1), (1, 5))
             for stride in ((8, 1), (8, 2), (4, 1), (6, 1), (1, 8)) for off in (0, 1, 3, 5, 11)]
    ids = torch.arange(64)
    cells = [set(ids.as_strided(v.shape, v.stride(), v.storage_offset()).flatten().tolist()) for v in views]
    for (a, ca), (b, cb) in itertools.product(zip(views, cells), repeat=2):
        if ca & cb:
            assert may_overlap(a, b)


def test_in_place_shares_all_or_none():
    from eraserdit_b200._native import refuse_overlap
    buf = torch.zeros(6, 100)
    refuse_overlap("out", buf[:, :40], (buf[:, 40:],), buf[:, :40])
    with pytest.raises(ValueError):
        refuse_overlap("out", buf[:, :40], (), buf[:, 1:41])
    with pytest.raises(ValueError):
        refuse_overlap("out", buf[:, :40], (buf[:, 39:],))
