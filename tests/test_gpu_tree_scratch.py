"""What hxm_tree_attention keeps between its launches goes by the tokens that can be read: by the
window where there is one, not by the whole table; and results do not go by the table's width."""
import pytest
import torch

import hxm
import hxm.ops as ops
from test_gpu_tree_attention import build, check, trees

pytestmark = pytest.mark.gpu

MB = 1 << 20


def taken(f):
    """Device memory that the library holds more of after f() than after releasing everything."""
    f()
    torch.cuda.synchronize()
    hxm.check(hxm.lib.hxm_release_cache(), "hxm_release_cache")
    free = torch.cuda.mem_get_info()[0]
    f()
    torch.cuda.synchronize()
    return free - torch.cuda.mem_get_info()[0]


# Heads times tiles of 128 rows of D + 2 floats: pieces that the tokens can make, and 2 MiB, a
# step of the device's allocator, twice.
@pytest.mark.parametrize("B,T,hkv,group,dim,page,table_pages,window,most", [
    (5, 25, 1, 12, 64, 32, 512, 1000, 75 * 128 * 66 * 4),     # 9 units of 128 tokens: 5 pieces
    (4, 64, 8, 4, 128, 64, 512, 0, 512 * 128 * 130 * 4),      # as many pieces as run at once
    (3, 9, 2, 4, 128, 16, 2048, 480, 0),                      # never cut
])
def test_memory_taken(dev, B, T, hkv, group, dim, page, table_pages, window, most):
    kc = torch.zeros(2, hkv, page, dim, dtype=torch.float16, device=dev)
    q = torch.zeros(B, T, hkv * group, dim, dtype=torch.float16, device=dev)
    table = torch.zeros(B, table_pages, dtype=torch.int32, device=dev)
    lens = torch.full((B,), page * table_pages - 1, dtype=torch.int32, device=dev)
    out = torch.empty_like(q)
    got = taken(lambda: ops.tree_attention(q, kc, kc.clone(), table, lens, window=window, out=out))
    assert got <= most + 4 * MB, f"{got / MB:.1f} MiB"


@pytest.mark.parametrize("window", [1, 100, 470])
def test_a_window_that_is_never_cut_needs_no_call_before_its_capture(dev, window):
    """Of sequences that are read up to 512 tokens each there is nothing to keep."""
    g = torch.Generator().manual_seed(window)
    lens, T = [1500, 9, 800], 9
    rows = trees(g, lens, T, "full")
    q, kc, vc, table, ld, seqs = build(g, "f16", lens, T, rows, 2, 4, 64, 16, "hnd", dev)
    qd, parents = q.to(dev), torch.tensor(rows, dtype=torch.int32, device=dev)
    out, lse = ops.tree_attention(qd, kc, vc, table, ld, parents, window=window, return_lse=True)
    check(out.cpu(), lse.cpu(), q, seqs, rows, 4, 64 ** -0.5, window, "f16")
    torch.cuda.synchronize()
    hxm.check(hxm.lib.hxm_release_cache(), "hxm_release_cache")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got, refused = torch.zeros_like(out), None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got.zero_()
        try:
            ops.tree_attention(qd, kc, vc, table, ld, parents, window=window, out=got)
        except hxm.HxmError as e:
            refused = e
    assert refused is None, refused
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, out)
        ops.tree_attention(qd, kc, vc, table, ld, parents, out=torch.empty_like(out))
        torch.cuda.synchronize()


@pytest.mark.parametrize("window", [470, 481, 482, 513, 1000, 2100])
@pytest.mark.parametrize("T,group", [(4, 4), (12, 4), (33, 6)])
def test_results_do_not_go_by_the_tables_width(dev, window, T, group):
    """Windows on both sides of what is cut, in a table of the sequences' pages and in one of
    2^20 tokens: the same bits, and right."""
    g = torch.Generator().manual_seed(window + T)
    lens = [2500, T, 0, 1037, 481 + T, 700]
    rows = trees(g, lens, T, "ragged")
    q, kc, vc, table, ld, seqs = build(g, "bf16", lens, T, rows, 1, group, 64, 16, "nhd", dev)
    qd, parents = q.to(dev), torch.tensor(rows, dtype=torch.int32, device=dev)
    out, lse = ops.tree_attention(qd, kc, vc, table, ld, parents, window=window, return_lse=True)
    check(out.cpu(), lse.cpu(), q, seqs, rows, group, 64 ** -0.5, window, "bf16")
    wide = torch.full((len(lens), 1 << 16), -1, dtype=torch.int32, device=dev)
    wide[:, :table.shape[1]] = table
    again = ops.tree_attention(qd, kc, vc, wide, ld, parents, window=window, return_lse=True)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
