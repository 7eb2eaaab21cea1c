"""Attention over shared pages where not all entities of many rows find room for images of their pages: those that do have them, the others are served without, and all alike within the bound."""
import ctypes as C

import numpy as np
import pytest

from test_gpu_pages_shared import LONG, MANY, attention, close, queries, run
from test_gpu_sequences import Cache, ints, starts, status_is_clear  # noqa: F401
from test_sequences_cpu import struct

pytestmark = pytest.mark.gpu
GROUP = 8                       # query heads of a kv head
NEW = -(-MANY // GROUP)         # tokens that make a sequence one of many rows


def room_for(gpu, n_pages, n_tok, stride, heads_kv, group=GROUP):
    """Bytes of the workspace, and of one page's image."""
    size = lambda n: gpu.lib().bonsai_b200_pages_attn_shared_workspace(  # noqa: E731
        C.byref(struct(n_pages=n, n_layers=1, n_head_kv=heads_kv, n_seq=1, table_stride=stride, n_tok=n_tok)), 0, group * heads_kv)
    return size(n_pages) - size(n_pages - 1)


def cache_of(gpu, n_pages, pages, new, heads_kv, seed=0):
    """Sequences of so many pages each, drawn from a pool of n_pages: they share them by their tables, without being a group."""
    c = Cache(gpu, [64 * n_pages], [sum(new)], n_head_kv=heads_kv, seed=seed, spare=0)
    rng = np.random.default_rng(seed)
    c.new, c.start = list(new), starts(new)
    c.lens = [64 * p - int(rng.integers(0, 64 - 1)) for p in pages]
    c.table = np.full((len(pages), max(pages)), -1, np.int32)
    for s, p in enumerate(pages):
        c.table[s, :p] = rng.integers(0, n_pages, p)
    c.view = gpu.Pages(c.d_pool, ints(c.table), ints(c.lens), ints(c.start), 1, heads_kv, c.n_tok)
    c.group, c.shared = ints([]), ints([])
    return c


@pytest.mark.parametrize("n_pages,pages,new,images", [
    (75, [80, 40, 60, LONG, 35], [NEW] * 5, [0, 40, 0, LONG, 0]),            # one larger than all the room, in front; one too many; one that fits; one more
    (100, [60, 60, 40, 2, 33], [NEW, NEW, NEW, 1, NEW], [60, 0, 40, 0, 0]),
    (64, [64, LONG, LONG], [NEW, NEW, NEW], [64, 0, 0]), (64, [LONG, 64, LONG], [NEW, NEW, NEW], [LONG, 0, LONG]),
    (90, [40, 40], [NEW, NEW - 1], [40, 0]), (40, [39, 40, 41], [1, NEW, NEW], [0, 40, 0]),
    # the ones that find none in front of many others: more entities than are looked at at once
    (70, [71, LONG] + [1] * 520 + [71, LONG, LONG], [NEW, NEW] + [1] * 520 + [NEW, NEW, NEW], [0, LONG] + [0] * 521 + [LONG, 0])])
@pytest.mark.parametrize("heads_kv", [4, 5])
def test_images_for_those_that_fit(gpu, n_pages, pages, new, images, heads_kv):
    import torch
    c = cache_of(gpu, n_pages, pages, new, heads_kv, seed=n_pages)
    q = queries(c, GROUP * heads_kv)
    want, most = attention(c, q)
    close(run(c, q), want, most)
    # which pages have images: their places one after the other from the workspace's begin on
    each = room_for(gpu, n_pages, c.n_tok, max(pages), heads_kv)
    ws = torch.full((c.view.attn_shared_workspace(0, GROUP * heads_kv),), 0xA5, dtype=torch.uint8, device="cuda")
    out = torch.full_like(q, 7.0)
    assert c.view.attn_shared(0, None, None, q, out, GROUP * heads_kv, ws, 0.0625) == 0
    written = (ws[:n_pages * each].reshape(n_pages, heads_kv, -1) != 0xA5).any(-1).all(-1)
    untouched = (ws[:n_pages * each].reshape(n_pages, -1) == 0xA5).all(-1)
    n = sum(images)
    assert bool(written[:n].all()) and bool(untouched[n:].all()), (n, int(written.sum()))
    close(out, want, most)


def test_a_captured_call_with_other_lengths(gpu):
    """The same graph, whose sequences fit or do not by their lengths when it is replayed."""
    import torch
    c = cache_of(gpu, 64, [64, LONG, 40], [NEW] * 3, 4, seed=9)
    q = queries(c, 4 * GROUP)
    ws, out = torch.empty(c.view.attn_shared_workspace(0, 4 * GROUP), dtype=torch.uint8, device="cuda"), torch.empty_like(q)
    step = lambda: c.view.attn_shared(0, None, None, q, out, 4 * GROUP, ws, 0.0625)  # noqa: E731
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(st):
        assert step() == 0
        with torch.cuda.graph(graph, stream=st):
            assert step() == 0
    torch.cuda.synchronize()
    rng = np.random.default_rng(1)
    c.table[:] = rng.integers(0, 64, c.table.shape)
    c.view._keep[1].copy_(ints(c.table))
    for lens in ([64 * 64, 64 * LONG, 64 * 40], [64 * 40, 64 * LONG, 64 * 33], [100, 64 * 64, 64 * LONG], [64 * LONG, 64 * LONG - 3, 90]):
        c.lens = lens
        c.view._keep[2].copy_(ints(lens))
        got = []
        for call in (graph.replay, step):
            out.fill_(7.0)
            ws.fill_(0xFF)
            call()
            torch.cuda.synchronize()
            got.append(out.clone())
        assert torch.equal(*got)
        close(out, *attention(c, q))
