"""hxm_tree_attention: a padded node, and a sequence without tokens, give zeros and -inf
whatever else is wrong with them; NaN are the others'."""
import numpy as np
import pytest
import torch

import hxm.ops as ops

pytestmark = pytest.mark.gpu

# T x group: one, two and four waves over the rows of a key head.
SHAPES = [(5, 2), (10, 6), (20, 5)]


def inputs(dev, B, T, group, table_pages, dim=64, hkv=2, page=16, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).half().to(dev)                   # noqa: E731
    table = torch.arange(B * table_pages, dtype=torch.int32, device=dev).view(B, table_pages)
    return (r(B, T, hkv * group, dim), r(B * table_pages, hkv, page, dim),
            r(B * table_pages, hkv, page, dim), table)


def call(dev, q, kc, vc, table, lens, rows):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)               # noqa: E731
    out, lse = ops.tree_attention(q, kc, vc, table, i32(lens), i32(rows), return_lse=True)
    return out.cpu(), lse.cpu()


def empty(out, lse):
    return bool((out == 0).all()) and bool((lse == -np.inf).all())


@pytest.mark.parametrize("T,group", SHAPES)
@pytest.mark.parametrize("table_pages", [4, 40])      # uncut sequences, and those that may be cut
def test_no_tokens_whatever_the_parents(dev, T, group, table_pages):
    """The parents of a sequence of the batch's padding are what an earlier step left."""
    q, kc, vc, table = inputs(dev, 5, T, group, table_pages)
    rows = [list(range(-1, T - 1)),
            [T - 1] * T,                              # later nodes
            list(range(T)),                           # themselves
            [-1, -2] + [1] * (T - 2),                 # below padding
            [2 ** 31 - 1] + [-2 ** 31] * (T - 1)]
    out, lse = call(dev, q, kc, vc, table, [60, 0, 0, -1, -2 ** 31], rows)
    assert out[0].isfinite().all() and lse[0].isfinite().all()
    for b in range(1, 5):
        assert empty(out[b], lse[b]), b


@pytest.mark.parametrize("T,group", SHAPES)
@pytest.mark.parametrize("table_pages", [4, 40])
def test_padding_of_a_sequence_of_a_wrong_length(dev, T, group, table_pages):
    """Too few tokens for the nodes, or more than the table holds: NaN, but for the padding."""
    q, kc, vc, table = inputs(dev, 4, T, group, table_pages)
    row = [-1, 0, -2, 1] + [-3] * (T - 4)
    lens = [T - 1, 1, 16 * table_pages + 1, 2 ** 31 - 1]
    out, lse = call(dev, q, kc, vc, table, lens, [row] * 4)
    live = [i for i, p in enumerate(row) if p >= -1]
    pads = [i for i, p in enumerate(row) if p < -1]
    for b in range(4):
        assert out[b, live].isnan().all() and lse[b, live].isnan().all(), b
        assert empty(out[b, pads], lse[b, pads]), b
