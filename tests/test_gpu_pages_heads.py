"""Attention over shared pages with few kv heads: which form a call takes goes by the rows and pages of all of them.  Each side of the borders against 64 bits, and which side it was, by the
images that a call leaves in its workspace."""
import pytest

from captured import capture
from test_gpu_pages_room import room_for
from test_gpu_pages_shared import attention, close, queries, run, shared_cache
from test_gpu_sequences import status_is_clear  # noqa: F401

pytestmark = pytest.mark.gpu
CASES = [  # kv heads, query heads of each, tokens, pages in common, whether they are written down as images
    (1, 1, 1025, 93, True), (1, 1, 1024, 93, False), (1, 1, 1025, 92, False), (1, 24, 86, 47, True), (1, 24, 86, 46, False), (1, 64, 33, 45, True), (1, 200, 11, 44, True),
    (2, 1, 1025, 32, True), (2, 1, 1025, 31, False), (2, 1, 641, 38, True), (2, 1, 641, 37, False), (2, 8, 129, 32, True), (3, 1, 641, 32, True), (3, 1, 640, 43, False), (3, 4, 171, 31, False),
    (4, 1, 641, 32, True), (4, 1, 640, 32, False), (6, 1, 641, 31, False)]


@pytest.mark.parametrize("each,heads_kv,group,n_tok,pages,images", [(each, *c) for c in CASES for each in (["many sequences", "two prompts"] if c[-1] else ["two prompts"])])
def test_borders(gpu, each, heads_kv, group, n_tok, pages, images):
    import torch
    if each == "two prompts":
        new, cached = [n_tok // 2, n_tok - n_tok // 2], [0, 70]
    else:
        n = min(n_tok, 40)
        new, cached = [n_tok // n + (i < n_tok % n) for i in range(n)], [i % 9 for i in range(n)]
    c = shared_cache(gpu, [len(new)], [pages], cached, new, n_head_kv=heads_kv, seed=n_tok)
    n_head = heads_kv * group
    q = queries(c, n_head)
    want, most = attention(c, q)
    close(run(c, q), want, most)
    ws = torch.full((c.view.attn_shared_workspace(1, n_head),), 0xA5, dtype=torch.uint8, device="cuda")
    out = torch.full_like(q, 7.0)
    call = lambda: c.view.attn_shared(0, c.group, c.shared, q, out, n_head, ws, 0.0625)  # noqa: E731
    assert call() == 0
    # a call whose rows could not be so many has no launches for images: a plan, the products, a join
    graph, kernels, _ = capture(call)
    enough = n_tok * group > 640 and n_tok * n_head > 1024
    assert graph is not None and len(kernels) == (5 if enough else 3)
    ws.fill_(0xA5)
    graph.replay()
    close(out, want, most)
    if n_tok * group > 640:                         # (fewer rows: there is no room)
        each_page = room_for(gpu, 100, n_tok, 200, heads_kv, group)
        written = (ws[:each_page * pages].reshape(pages, -1) != 0xA5).any(-1)
        assert bool(written.all()) if images else not enough or not bool((ws[:1024] != 0xA5).any())
