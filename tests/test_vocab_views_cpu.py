"""Which views the vocabulary operators take as outputs: what shares no element with an input is taken. Host code
alone, no GPU needed."""
import random

import pytest
import torch

from raft_b200 import linalg


def elements(t):
    """The addresses of a tensor's elements, one by one."""
    at = torch.zeros(t.shape, dtype=torch.int64)
    for d, (n, s) in enumerate(zip(t.shape, t.stride())):
        at += (torch.arange(n) * s).view([-1 if i == d else 1 for i in range(t.dim())])
    return set((t.data_ptr() + at.reshape(-1) * t.element_size()).tolist())


def test_column_blocks_of_one_buffer_do_not_overlap():
    wide = torch.zeros((6, 20))
    assert not linalg._overlap(wide[:, :10], wide[:, 10:])
    assert not linalg._overlap(wide[:, 12:], wide[:, :12])
    assert linalg._overlap(wide[:, :11], wide[:, 10:])
    assert linalg._overlap(wide, wide[2, 5:7])
    assert not linalg._overlap(wide[:, :10], wide[2, 10:20])  # a vector between two rows
    assert linalg._overlap(wide[:, :10], wide.view(-1)[30:41])
    assert not linalg._overlap(wide[:, :10], wide.view(-1)[30:40])


@pytest.mark.parametrize("seed", range(40))
def test_overlap_is_what_the_elements_say(seed):
    """Matrices of rows at the same or at different strides and vectors, laid over one buffer at random."""
    rng = random.Random(seed)
    base = torch.zeros(200)
    both = {True: 0, False: 0}

    def some():
        rows, cols = rng.choice([1, 2, 3, 5]), rng.randint(1, 12)
        stride = rng.choice([cols, cols + 1, cols + 5, 31, 31])
        at = rng.randint(0, 200 - ((rows - 1) * stride + cols))
        return base.as_strided((rows, cols), (stride, 1), at)
    for _ in range(60):
        a, b = some(), some()
        want = bool(elements(a) & elements(b))
        assert linalg._overlap(a, b) == linalg._overlap(b, a) == want, (a.shape, a.stride(), b.shape, b.stride())
        both[want] += 1
    assert min(both.values()) > 0


def test_overlap_of_other_shapes_and_types():
    raw = torch.zeros(4096, dtype=torch.uint8)
    halves = raw.view(torch.float16).view(4, 8, 64)
    assert linalg._overlap(halves, raw[4000:].view(torch.int32))
    column = raw.view(torch.int64)[:96].view(12, 8)[:, 2:3]  # a column: rows of one element
    assert not linalg._overlap(column, raw.view(torch.int64)[3:10])
    assert linalg._overlap(column, raw.view(torch.int64)[3:11])
    assert not linalg._overlap(halves[:0], halves) and not linalg._overlap(halves, raw[:0])


def test_other_layouts_count_with_what_they_span():
    base = torch.zeros(100)
    assert linalg._overlap(base[:50:2], base[1:50:2]) and not linalg._overlap(base[:50:2], base[50:])
    assert linalg._overlap(base[:10].expand(5, 10), base[9:20]) and not linalg._overlap(base[:10].expand(5, 10), base[10:])
    assert linalg._overlap(base.view(10, 10).t()[:3], base[90:]) and not linalg._overlap(base.view(10, 10).t()[:, :3], base[30:])
