"""Cache rows written by CTAs of two tokens (calls of many rows): an odd last token, two sequences in a CTA, several groups of rows, queries in their own place, replayed graphs.  Which form a
call takes is read from what it launches, so that cases which no longer reach this one are noticed."""
import numpy as np
import pytest

from captured import capture
from test_gpu_rotary_and_rows import test_write as check_write
from test_gpu_sequences import Cache, ints, starts, status_is_clear  # noqa: F401

pytestmark = pytest.mark.gpu
CASES = {  # lengths, new tokens, query heads, kv heads, rows of nobody
    "several sequences, ends at odd rows, an odd last token": ([300, 64, 1, 0, 461], [201, 2, 1, 0, 397], 24, 4, 0),
    "a last CTA with one token and none": ([700], [600], 24, 4, 1),
    "rows of nobody in a CTA with somebody's": ([65, 640], [1, 600], 24, 4, 4),
    "two groups of rows, the second a short one": ([130, 200], [130, 111], 70, 2, 0),
    "three groups, no queries but one": ([1, 190], [1, 160], 1, 66, 0),
    "two sequences in every CTA": ([1 + 7 * i % 64 for i in range(601)], [1] * 601, 22, 2, 0),
    "keys and values only": ([500, 500], [399, 500], 0, 9, 0)}


def grid(call):
    """Of the one kernel that a call launches."""
    from cuda.bindings import driver
    graph, kernels, _ = capture(call)      # (the nodes are the graph's: it has to stay)
    assert len(kernels) == 1
    err, params = driver.cuGraphKernelNodeGetParams(driver.CUgraphNode(init_value=int(kernels[0])))
    assert int(err) == 0 and graph is not None
    return params.gridDimX, params.gridDimY


def two_tokens(n_tok, rows):
    return (n_tok + 1) // 2, -(-rows // 64)


@pytest.mark.parametrize("case", CASES)
def test_form(gpu, case):
    import torch
    lens, new, n_head, n_head_kv, behind = CASES[case]
    c = Cache(gpu, lens, new, n_head_kv=n_head_kv, behind=behind)
    q, k, v = (torch.zeros(c.n_tok, h, 256, device="cuda") for h in (n_head, n_head_kv, n_head_kv))
    wide = n_head * 256, 256, n_head_kv * 256, 256, n_head_kv * 256, 256
    assert grid(lambda: c.view.write(0, q, k, v, None, None, None, None, torch.empty_like(q), n_head, 0, 0, 1.0, *wide, 1e-6)) == two_tokens(c.n_tok, n_head + 2 * n_head_kv)


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("n_rot,pairs,norm", [(64, 0, True), (256, 1, True), (62, 0, False), (6, 1, True)])
@pytest.mark.parametrize("layout", ["packed", "beside a gate", "odd"])
def test_rows(gpu, case, n_rot, pairs, norm, layout):
    """Queries, bytes, and every other byte as it was."""
    check_write(gpu, *CASES[case], n_rot, pairs, norm, layout)


@pytest.mark.parametrize("pairs", [0, 1])
@pytest.mark.parametrize("odd", [0, 1])
def test_write_is_rope_and_append(gpu, pairs, odd):
    """Bit for bit, without norms; queries in the place of the projection."""
    import torch
    a, b = (Cache(gpu, [700, 70], [598, 3], seed=4) for _ in range(2))
    n = a.n_tok
    q, k, v = (torch.randn(n * h * 256 + odd, device="cuda")[odd:].reshape(n, h, 256) for h in (24, 4, 4))
    freq, amplitude = gpu.rope_freq(64, 1e7, "yarn", 4.0, 262144)
    freq = freq.cuda()
    pos = torch.cat([torch.arange(102, 700), torch.arange(67, 70)]).int().cuda()
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    assert gpu.rope(q, k, pos, freq, q_out, k_out, n, 24, 4, 256, 64, pairs, amplitude, 6144, 256, 1024, 256) == 0
    assert a.view.append(0, k_out, v) == 0
    write = lambda out: b.view.write(0, q, k, v, None, None, None, freq, out, 24, 64, pairs, amplitude, 6144, 256, 1024, 256, 1024, 256, 1e-6)  # noqa: E731
    assert grid(lambda: write(torch.empty_like(q))) == two_tokens(n, 32)
    b.upload()
    assert write(q) == 0
    assert torch.equal(q, q_out) and torch.equal(a.d_pool, b.d_pool)


def test_captured_rows_follow_the_numbers(gpu):
    """A captured call is replayed with other lengths and rows, some of them nobody's; the call by itself on another stream."""
    import torch
    c = Cache(gpu, [900, 300], [601, 3], seed=11, spare=20)
    n = c.n_tok
    q, k, v = (torch.randn(n, h, 256, device="cuda") for h in (24, 4, 4))
    w, freq, out = torch.rand(256, device="cuda"), gpu.rope_freq(64, 1e7)[0].cuda(), torch.empty_like(q)
    step = lambda: c.view.write(0, q, k, v, w, w, None, freq, out, 24, 64, 0, 1.0, 6144, 256, 1024, 256, 1024, 256, 1e-6)  # noqa: E731
    graph, kernels, _ = capture(step)
    assert len(kernels) == 1 and grid(step) == two_tokens(n, 32)
    torch.cuda.synchronize()
    length, start = c.view._keep[2:]
    for lens, new in (([704, 301], [4, 1]), ([640, 64], [0, 64]), ([604, 1], [603, 1]), ([601, 3], [601, 3]), ([333, 271], [333, 271])):
        length.copy_(ints(lens))
        start.copy_(ints(starts(new)))
        got = []
        for run in (graph.replay, step):
            c.upload()
            out.fill_(7.0)
            run()
            torch.cuda.synchronize()
            got.append((out.clone(), c.d_pool.clone()))
        assert all(torch.equal(a, b) for a, b in zip(*got))
        assert bool((got[0][0][sum(new):] == 7).all()) and not bool((got[0][0][:sum(new)] == 7).all(-1).any())
        # a token at a time, by the other form: the same bits
        c.upload()
        for s in range(2):
            for t in range(0, new[s], 50):
                m = min(50, new[s] - t)
                rows = slice(start[s].item() + t, start[s].item() + t + m)
                own = gpu.Pages(c.d_pool, ints(c.table[s:s + 1]), ints([lens[s] - new[s] + t + m]), ints([0, m]), 1, 4, m)
                few = torch.empty(m, 24, 256, device="cuda")
                assert own.write(0, q[rows], k[rows], v[rows], w, w, None, freq, few, 24, 64, 0, 1.0, 6144, 256, 1024, 256, 1024, 256, 1e-6) == 0
                assert torch.equal(few, got[0][0][rows])
        assert torch.equal(c.d_pool, got[0][1])


def test_places_that_do_not_fit(gpu):
    """A page that the pool does not have, and more new tokens than positions: that sequence's rows, in whichever half of a CTA, and no others."""
    import torch
    c = Cache(gpu, [300, 5, 460], [201, 5, 397], seed=10)
    q, k, v = (torch.randn(c.n_tok, h, 256, device="cuda") for h in (24, 4, 4))
    step = lambda out: c.view.write(0, q, k, v, None, None, None, None, out, 24, 0, 0, 1.0, 6144, 256, 1024, 256, 1024, 256, 1e-6)  # noqa: E731
    assert grid(lambda: step(torch.empty_like(q))) == two_tokens(c.n_tok, 32)
    c.upload()
    assert step(torch.empty_like(q)) == 0
    whole = c.d_pool.clone()
    for at, value, gone in ((1, c.n_pages, range(201, 206)), (2, 3, (201, 202))):
        c.view._keep[at].copy_(ints(c.table if at == 1 else c.lens))
        c.view._keep[at][(1, 0) if at == 1 else 1] = value
        c.upload()
        out = torch.full_like(q, 7.0)
        assert step(out) == 0
        assert gpu.device_status() == 3 and gpu.clear_status() == 0
        kept = torch.ones(c.n_tok, dtype=torch.bool, device="cuda")
        kept[list(gone)] = False
        assert torch.equal(out[kept], q[kept]) and bool((out[~kept] == 7).all())
        others = torch.ones(c.n_pages, dtype=torch.bool, device="cuda")
        others[int(c.table[1, 0])] = False
        assert torch.equal(c.d_pool[others], whole[others])
        c.view._keep[at].copy_(ints(c.table if at == 1 else c.lens))
