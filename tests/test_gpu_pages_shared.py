"""Attention over pages that sequences share, by both of its kernels, against a plain statement in 64 bits; and a step of all calls around such a cache."""
import math

import numpy as np
import pytest

from test_gpu_pages_division import attention as plain_attention, queries
from test_gpu_sequences import U, Cache, ints, number, run_attention, starts, status_is_clear  # noqa: F401

pytestmark = pytest.mark.gpu
MANY, LONG = 641, 32            # rows and pages from which on the pages of an entity are written down as images


# Roundings, in u of size = (1 + largest |q k| of a row) times sum of p |v|.  A score: planes' products without low times low 4, 48 matrix instructions that cut their sums off at
# 2^-23 of them 96 and the lift against that 12, factors 5, less its reference 2.  A weight: 2^x 4, planes 5.  An output: planes' products 4, 24 matrix instructions a step 48, and a step's
# sum, its change of reference and its part of a join 3 for each page; the sum of weights the same 3, division and product 3.
# Planes of weights are fp16: what both leave of a weight is 2^-22 of it (half of 2^-11, of half of 2^-11) or half of fp16's smallest step, 2^-25, if that is more.  A row's largest weight is 2^7
# at least, and their sum with it: 2^-32 of the sum of |v| of all positions that are seen.
def attention(c, q, layer=0, scale=0.0625):
    """Outputs in 64 bits, and what they may be off by."""
    import torch
    want, size = plain_attention(c, q, layer=layer, scale=scale)
    seen = torch.zeros_like(size)
    group = q.shape[1] // c.hkv
    for s, n in enumerate(c.new):
        length = c.lens[s]
        for j in range(c.hkv if n and length else 0):
            v = torch.from_numpy(number(c.pool[c.table[s, :-(-length // 64)], layer, 1, j].reshape(-1, 8, 34)[:length])).cuda().abs().cumsum(0)
            seen[c.start[s]:c.start[s] + n, j * group:(j + 1) * group] = v[length - n:, None]
    return want, size * U * (190 + 6 * -(-max(c.lens) // 64)) + 2.0 ** -32 * seen


def shared_cache(gpu, groups, shared, cached, new, alone=0, **kw):
    """groups: sequences of each; shared: pages of each; cached, new: of each sequence behind what it shares.  The last `alone` sequences are of no group."""
    first = starts(groups)
    of = [g for g, n in enumerate(groups) for _ in range(n)] + [-1] * alone
    lens = [(shared[g] * 64 if g >= 0 else 0) + c + n for g, c, n in zip(of, cached, new)]
    c = Cache(gpu, lens, new, **kw)
    for s, g in enumerate(of):
        if g >= 0:
            c.table[s, :shared[g]] = c.table[first[g], :shared[g]]
    c.view._keep[1].copy_(ints(c.table))
    c.group, c.shared, c.of = ints(first), ints(shared), of
    return c


def run(c, q, layer=0, scale=0.0625, out=None):
    """With a workspace of exactly the bytes asked for, 4 KB of marks on either side of it and of the outputs."""
    import torch
    size, n, groups = c.view.attn_shared_workspace(len(c.shared), q.shape[1]), q.numel(), len(c.shared)
    room = torch.full((size + 8192,), 0xA5, dtype=torch.uint8, device="cuda")
    room[4096:4096 + size].view(torch.float32).fill_(math.nan)
    outs = torch.full((n + 2048,), 7.0, device="cuda")
    out = outs[1024:1024 + n].reshape(q.shape)
    pool = c.d_pool.clone()
    assert c.view.attn_shared(layer, c.group if groups else None, c.shared if groups else None, q, out, q.shape[1], room[4096:4096 + size], scale) == 0
    assert bool((room[:4096] == 0xA5).all()) and bool((room[4096 + size:] == 0xA5).all())
    assert bool((outs[:1024] == 7).all()) and bool((outs[1024 + n:] == 7).all()) and torch.equal(pool, c.d_pool)
    return out


def close(got, want, most):
    off = (got.double() - want).abs()
    assert bool((off <= most).all()), f"{(off / most.clamp(min=1e-300)).max().item():.2f} of the bound"


CASES = [  # sequences of the groups, pages in common, cached and new tokens of each sequence, sequences alone, query heads, kv heads, rows of nobody
    ([1], [0], [0], [1], 0, 24, 4, 0), ([2], [1], [0, 0], [1, 1], 0, 24, 4, 0), ([2], [1], [63, 0], [1, 2], 0, 24, 4, 3), ([2], [2], [64, 65], [1, 1], 0, 24, 4, 0),
    ([2], [3], [0, 0], [1, 0], 0, 24, 4, 0), ([3], [3], [1, 2, 3], [0, 0, 1], 0, 24, 4, 2), ([1], [5], [10], [3], 0, 24, 4, 0), ([], [], [100, 0, 3], [1, 7, 0], 3, 24, 4, 1),
    ([8], [5], [0, 1, 63, 64, 65, 128, 200, 31], [1] * 8, 0, 24, 4, 0), ([9], [4], [i * 17 for i in range(9)], [1] * 9, 0, 24, 4, 0),
    ([3, 0, 2, 1], [2, 9, 1, 4], [10, 20, 30, 0, 100, 5], [1, 2, 3, 4, 5, 6], 0, 24, 4, 0), ([2, 3], [2, 0], [5, 6, 7, 80, 9, 300, 0], [1, 30, 1, 1, 2, 1, 50], 2, 24, 4, 4),
    ([4], [7], [0, 5, 9, 200], [5, 5, 5, 5], 0, 24, 4, 0), ([4], [3], [0, 64, 0, 1], [100, 64, 3, 1], 0, 8, 8, 0), ([40], [6], [i for i in range(40)], [1] * 40, 0, 8, 1, 0),
    ([5], [4], [3] * 5, [2] * 5, 0, 5, 1, 0), ([3], [2], [70, 0, 1], [1, 1, 1], 0, 64, 64, 0), ([2], [2], [0, 9], [3, 2], 0, 200, 1, 0), ([2], [2], [0, 9], [1, 2], 0, 6, 6, 0),
    ([12, 5], [LONG, 10], [0] * 17, [9] * 12 + [1] * 5, 0, 24, 4, 0),                                   # 648 rows over 32 pages: images
    ([2], [LONG], [0, 100], [100, 7], 0, 24, 4, 1),                                                     # 642
    ([2], [LONG - 1], [0, 100], [100, 7], 0, 24, 4, 0), ([2], [LONG], [0, 100], [99, 7], 0, 24, 4, 0),      # a page, a token fewer
    ([27], [LONG + 3], [3 * i for i in range(27)], [1] * 27, 0, 24, 1, 0), ([3], [LONG], [5, 0, 0], [300, 301, 50], 0, 2, 2, 0), ([2, 2], [40, 33], [0, 1, 2, 3], [60, 60, 60, 50], 0, 24, 4, 0),
    ([1], [0], [2100], [200], 0, 24, 4, 0), ([], [], [2048, 3], [641, 2], 2, 4, 4, 0),                  # a prompt by itself: images of its own pages, rows that see to their own
    ([2], [35], [2000, 0], [130, 20], 0, 24, 4, 2), ([3], [33], [1, 0, 5], [200, 0, 140], 0, 8, 2, 0), ([4], [LONG], [0] * 4, [170, 1, 1, 1], 0, 16, 4, 0), ([2], [64], [0, 0], [6, 5], 0, 64, 1, 0)]


@pytest.mark.parametrize("groups,shared,cached,new,alone,n_head,n_head_kv,behind", CASES)
def test_attention(gpu, groups, shared, cached, new, alone, n_head, n_head_kv, behind):
    c = shared_cache(gpu, groups, shared, cached, new, alone, n_layers=2, n_head_kv=n_head_kv, behind=behind, seed=sum(cached))
    q = queries(c, n_head)
    want, most = attention(c, q, layer=1)
    close(run(c, q, layer=1), want, most)


@pytest.mark.parametrize("groups,shared,each,n_head", [([600], [3], 1, 8), ([300, 300], [40, 2], 1, 4), ([2] * 260, [1] * 260, 1, 4), ([40], [70], 2, 24)])
def test_many_sequences(gpu, groups, shared, each, n_head):
    rng = np.random.default_rng(len(groups))
    n = sum(groups)
    new = [0 if i % 7 == 3 else each for i in range(n)]
    c = shared_cache(gpu, groups, shared, rng.integers(0, 100, n).tolist(), new, n_head_kv=n_head // 4, seed=n)
    q = queries(c, n_head)
    want, most = attention(c, q)
    close(run(c, q), want, most)


FORMS = {"few rows": ([3, 2], [5, 2], [10, 0, 130, 64, 7], [1, 4, 2, 1, 1]), "many rows": ([3, 2], [40, 2], [10, 0, 130, 64, 7], [60, 40, 20, 1, 1])}


def cache_of(gpu, form, **kw):
    return shared_cache(gpu, *FORMS[form], **{"seed": 3, **kw})


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("scale", [-0.0625, 0.0, 1.0, 3.0])
def test_other_scales(gpu, form, scale):
    """Scores turned round, all the same, and far apart: weights of 0 and 1, references that move."""
    c = cache_of(gpu, form)
    q = queries(c, 24)
    want, most = attention(c, q, scale=scale)
    close(run(c, q, scale=scale), want, most)


@pytest.mark.parametrize("form", FORMS)
def test_scores_that_grow(gpu, form):
    """Later positions with larger keys: the reference of a row moves many times."""
    import torch
    c = cache_of(gpu, form, scale=0.02)
    q = queries(c, 24)
    for s, n in enumerate(c.lens):
        for p in range(-(-n // 64)):
            codes = c.pool[c.table[s, p], 0, 0].reshape(4, 64, 8, 34)
            d = codes[..., :2].copy().view(np.float16)
            codes[..., :2] = (np.abs(d) * 0 + np.float16(2.0 ** -12) * np.float16(1 + 3 * p)).astype(np.float16).view(np.uint8)
    c.upload()
    want, most = attention(c, q, scale=1.0)
    close(run(c, q, scale=1.0), want, most)
    assert torch.equal(run(c, q, scale=1.0), run(c, q, scale=1.0))


@pytest.mark.parametrize("form", FORMS)
def test_values_far_apart(gpu, form):
    """Scales of V (and of K's blocks) over 20 powers of two: exact all the same."""
    c = cache_of(gpu, form)
    q = queries(c, 24)
    rng = np.random.default_rng(9)
    flat = c.pool.reshape(-1, 8, 34)
    up = (2.0 ** rng.integers(-8, 9, (len(flat), 8, 1))).astype(np.float32)
    flat[..., :2] = (flat[..., :2].copy().view(np.float16).astype(np.float32) * up / 16).astype(np.float16).view(np.uint8)
    c.upload()
    want, most = attention(c, q, scale=0.001)
    close(run(c, q, scale=0.001), want, most)


@pytest.mark.parametrize("form", [*FORMS, "a prompt"])
@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("bits", [0x7E00, 0x7C00, 0xFC00])
def test_scales_that_are_no_numbers(gpu, form, kv, bits):
    """In the pages in common, and in a sequence's own: NaN for the tokens that see them, and for no others; in front of, at and behind the last position that a token sees."""
    import torch
    if form == "a prompt":
        c = shared_cache(gpu, [1], [0], [2000], [130], seed=8)
        marks = [(0, 2000, 0), (0, 2064, 1), (0, 2129, 2), (0, 2001, 3), (0, 2040, 3)]       # sequence, position, kv head
    else:
        c = cache_of(gpu, form)
        marks = [(4, 2 * 64 + 3, 2), (3, 70, 3)] if form == "few rows" else [(0, 40 * 64 + 11, 1), (2, 39 * 64 + 63, 2), (1, 40 * 64 + 30, 3), (1, 40 * 64 + 33, 3)]
    q = queries(c, 24)
    want, most = attention(c, q)
    bad = torch.zeros(c.n_tok, 24, dtype=torch.bool, device="cuda")
    for s, p, head in marks:
        c.pool[c.table[s, p // 64], 0, kv, head, p % 64].reshape(8, 34)[5, :2] = np.array([bits], np.uint16).view(np.uint8)
        common = p < 64 * c.shared.tolist()[c.of[s]]
        for t in range(len(c.new)):
            for i in range(c.new[t] if t == s or (common and c.of[t] == c.of[s]) else 0):
                if p <= c.lens[t] - c.new[t] + i:
                    bad[c.start[t] + i, head * 6:head * 6 + 6] = True
    c.upload()
    got = run(c, q)
    assert bool(bad.any()) and not bool(bad.all()) and bool(got[bad].isnan().all()) and not bool(got[~bad].isnan().any())
    close(got[~bad], want[~bad], most[~bad])


@pytest.mark.parametrize("form", FORMS)
def test_queries_that_are_no_numbers(gpu, form):
    """A NaN in a query counts as zero, an infinity makes that row no numbers, and no other; a query of zeros weighs everything alike."""
    import torch
    c = cache_of(gpu, form)
    q = queries(c, 24)
    q[3, 20], q[1, 7, 9], q[2, 3, 100] = 0.0, 0.0, 0.0
    want, most = attention(c, q)
    q[1, 7, 9], q[2, 3, 100] = math.nan, math.inf
    got = run(c, q)
    assert not bool(got[2, 3].isfinite().any())
    got[2, 3] = want[2, 3].float()
    close(got, want, most)


@pytest.mark.parametrize("form", FORMS)
def test_nothing_hidden_reaches_a_row(gpu, form):
    """Rows behind a token, of its own sequence and of pages that nobody is given: any bytes, the same bits."""
    import torch
    c = cache_of(gpu, form)
    q = queries(c, 24)
    want = run(c, q)
    held = np.zeros((c.n_pages, 64), bool)
    for s, n in enumerate(c.lens):
        for p in range(n):
            held[c.table[s, p // 64], p % 64] = True
    c.pool.transpose(0, 4, 1, 2, 3, 5, 6)[~held] = 0xFF     # NaN scales
    c.upload()
    assert torch.equal(run(c, q), want)


def test_tokens_without_a_position_see_nothing(gpu):
    c = Cache(gpu, [2, 40, 0], [5, 2, 3], seed=3)
    c.group, c.shared = ints([]), ints([])
    q = queries(c, 24)
    out = run(c, q)
    assert bool((out[:3] == 0).all()) and bool((out[7:] == 0).all())
    held = type("Held", (), {"n_tok": 4, "hkv": 4, "lens": [2, 40], "new": [2, 2], "start": [0, 2, 4], "pool": c.pool, "table": c.table})
    want, most = attention(held, q[3:7])
    close(out[3:7], want, most)


@pytest.mark.parametrize("form", FORMS)
def test_odd_offsets_and_other_attention(gpu, form):
    """Queries and outputs that begin 4 bytes behind 16: the same bits.  The attention that shares nothing: 1e-5 of the largest output of a head for each."""
    import torch
    c = cache_of(gpu, form)
    q = queries(c, 24)
    want = run(c, q)
    n = q.numel()
    qo, oo = torch.empty(n + 1, device="cuda"), torch.full((n + 2,), 7.0, device="cuda")
    qo[1:] = q.flatten()
    ws = torch.empty(c.view.attn_shared_workspace(2, 24), dtype=torch.uint8, device="cuda")
    assert c.view.attn_shared(0, c.group, c.shared, qo[1:].reshape(q.shape), oo[1:n + 1].reshape(q.shape), 24, ws, 0.0625) == 0
    assert torch.equal(oo[1:n + 1].reshape(q.shape), want) and oo[0].item() == 7 and oo[-1].item() == 7
    other = run_attention(gpu, c, q)
    assert bool(((want - other).abs() <= 2e-5 * other.abs().amax(-1, keepdim=True)).all())


@pytest.mark.parametrize("form", FORMS)
def test_numbers_that_do_not_fit(gpu, form):
    """Pages, lengths, rows and groups: what they concern is not served or incomplete, the rest within the bound, and the status word says so."""
    c = cache_of(gpu, form, spare=3)
    q = queries(c, 24)
    want, most = attention(c, q)
    table, length, start = c.view._keep[1:]
    rows = lambda *of: [r for s in of for r in range(c.start[s], c.start[s + 1])]  # noqa: E731

    def check(served, untouched=()):
        assert gpu.device_status() == 0
        out = run(c, q)
        assert gpu.device_status() == 3 and gpu.clear_status() == 0
        r = rows(*served)
        close(out[r], want[r], most[r])
        assert bool((out[rows(*untouched)] == 7).all())
    for page in (-1, c.n_pages, 2 ** 31 - 1, -2 ** 31):
        table[1, c.shared[0].item()] = page             # of a sequence's own
        check((0, 2, 3, 4))
        table.copy_(ints(c.table))
        table[0, 1] = page                              # in common: the first sequence's table is read
        check((3, 4))
        table.copy_(ints(c.table))
    for n in (table.shape[1] * 64 + 1, 2 ** 31 - 1, -1, 64, c.shared[0].item() * 64 + c.new[1] - 1):             # past the table, negative; new tokens among what is shared
        length[1] = n
        check((0, 2, 3, 4), (1,))
    length.copy_(ints(c.lens))
    for n in (table.shape[1] + 1, -1, 2 ** 31 - 1, -2 ** 31):
        c.shared[0] = n
        check((3, 4), (0, 1, 2))
    c.shared.copy_(ints(FORMS[form][1]))
    for first in ([0, 6, 5], [-1, 3, 5], [0, 2 ** 31 - 1, 5]):
        c.group.copy_(ints(first))
        run(c, q)
        assert gpu.device_status() == 3 and gpu.clear_status() == 0
    c.group.copy_(ints(starts(FORMS[form][0])))
    for at in ([0, 5, 3, c.start[3], c.start[4], c.start[5]], [0, 0, 0, 0, 0, c.n_tok + 1], [0, 2 ** 31 - 1, 2, 3, 4, 5], [-3, 1, 2, 3, 4, 5], [0, c.n_tok, 0, c.n_tok, 0, c.n_tok]):
        start.copy_(ints(at))
        run(c, q)
        assert gpu.device_status() == 3 and gpu.clear_status() == 0
    start.copy_(ints(c.start))
    close(run(c, q), want, most)


def test_captured_attention_follows_the_numbers(gpu):
    """A captured call is replayed with other rows, groups and numbers of pages in common: by one kernel or by both."""
    import torch
    c = cache_of(gpu, "many rows", spare=20)
    q, n = queries(c, 24), c.n_tok
    out = torch.empty_like(q)
    ws = torch.empty(c.view.attn_shared_workspace(2, 24), dtype=torch.uint8, device="cuda")
    step = lambda: c.view.attn_shared(0, c.group, c.shared, q, out, 24, ws, 0.0625)  # noqa: E731
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(st):
        assert step() == 0
        with torch.cuda.graph(graph, stream=st):
            assert step() == 0
    torch.cuda.synchronize()
    start, lens = c.view._keep[3], c.lens
    for group, shared, new in (([0, 3, 5], [40, 2], c.new), ([0, 3, 5], [40, 2], [1, 1, 1, 1, 1]), ([0, 2, 3], [38, 0], [50, 60, 0, 0, 1]), ([2, 3, 3], [1, 0], [0, 0, 0, 0, 0]),
                               ([0, 1, 3], [40, 38], [0, n - 3, 1, 1, 1])):
        c.group.copy_(ints(group))
        c.shared.copy_(ints(shared))
        start.copy_(ints(starts(new)))
        q.normal_()
        got = []
        for call in (graph.replay, step):
            out.fill_(7.0)
            ws.fill_(0xFF)
            call()
            torch.cuda.synchronize()
            got.append(out.clone())
        assert torch.equal(*got) and bool((out[sum(new):] == 7).all())
        held = type("Held", (), {"n_tok": n, "hkv": 4, "lens": lens, "new": new, "start": starts(new), "pool": c.pool, "table": c.table})
        want, most = attention(held, q)
        close(out, want, most)


@pytest.mark.parametrize("form", FORMS)
def test_other_streams_and_two_at_once(gpu, form):
    """The same bits on any stream, and of two calls with a workspace each that run over each other."""
    import torch
    made = []
    for i in range(2):
        c = cache_of(gpu, form, seed=40 + i)
        q = queries(c, 24, 50 + i)
        made.append((c, q, run(c, q), torch.cuda.Stream(), [torch.full_like(q, 7.0) for _ in range(4)], torch.empty(c.view.attn_shared_workspace(2, 24), dtype=torch.uint8, device="cuda")))
    torch.cuda.synchronize()
    for i in range(4):
        for c, q, _, stream, outs, ws in made:
            with torch.cuda.stream(stream):
                assert c.view.attn_shared(0, c.group, c.shared, q, outs[i], 24, ws, 0.0625) == 0
    torch.cuda.synchronize()
    for _, _, want, _, outs, _ in made:
        assert all(torch.equal(want, o) for o in outs)


def test_pages_far_into_a_pool(gpu):
    """A pool of more than 4 GB of which the last pages are used."""
    import torch
    for form in FORMS:
        c = cache_of(gpu, form)
        q = queries(c, 24)
        want = run(c, q)
        page = c.d_pool[0].numel()
        n = (1 << 32) // page + 2 + c.n_pages
        pool = torch.empty(n, page, dtype=torch.uint8, device="cuda")
        pool[n - c.n_pages:] = c.d_pool.reshape(c.n_pages, -1)
        table = ints(np.where(c.table >= 0, c.table + n - c.n_pages, -1))
        view = gpu.Pages(pool, table, *c.view._keep[2:], 1, 4, c.n_tok)
        ws, out = torch.empty(view.attn_shared_workspace(2, 24), dtype=torch.uint8, device="cuda"), torch.full_like(q, 7.0)
        assert view.attn_shared(0, c.group, c.shared, q, out, 24, ws, 0.0625) == 0
        assert torch.equal(out, want)
        # rows written and read there
        k, v = (torch.randn(c.n_tok, 4, 256, device="cuda") for _ in range(2))
        none = torch.empty(0, device="cuda")
        kr, vr, kw, vw = (torch.empty_like(k) for _ in range(4))
        for p, a, b in ((view, kr, vr), (c.view, kw, vw)):
            assert p.write(0, none, k, v, None, None, None, None, none, 0, 0, 0, 1.0, 0, 0, 1024, 256, 1024, 256, 1e-6) == 0 and p.read(0, None, a, b) == 0
        assert torch.equal(kr, kw) and torch.equal(vr, vw) and torch.equal(pool[n - c.n_pages:], c.d_pool.reshape(c.n_pages, -1))


def test_what_python_refuses(gpu, monkeypatch):
    import torch
    c = cache_of(gpu, "few rows")
    q = queries(c, 24)
    size = c.view.attn_shared_workspace(2, 24)
    ws, out = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.empty_like(q)
    args = dict(group=c.group, shared=c.shared, q=q, out=out, n_head=24, workspace=ws)
    call = lambda **bad: c.view.attn_shared(0, *{**args, **bad}.values(), 0.0625)  # noqa: E731
    assert call() == 0
    assert call(workspace=ws[:size - 16]) == 1 and call(workspace=None) == 1 and call(n_head=6) == 1
    for bad in ({"group": c.group[:2]}, {"q": q[:3]}, {"out": out[:3]}, {"shared": c.shared.long()}, {"group": c.group.float()}, {"q": q.half()}, {"q": q.cpu()}, {"n_head": 28}):
        with pytest.raises((RuntimeError, TypeError)):
            call(**bad)
    monkeypatch.setattr(c.view, "_device", c.view._device + 1)
    with pytest.raises(RuntimeError, match="the cache is on device"):
        call()


def test_a_step_of_all_calls(gpu):
    """A prompt is written and attended to once, answers go on from it by forks of its pages, each token attended to over what they share; the outputs are those of the attention that shares
    nothing.  Then the oldest page of one answer is dropped: what is left is read, turned back and written again, and attended to at its new positions."""
    import torch
    from bonsai_b200.pages import PageBook
    H, HKV, D, PAGES, PROMPT, N = 24, 4, 256, 64, 200, 5
    gen = torch.Generator(device="cuda").manual_seed(31)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    wq, wk = 1 + 0.1 * rand(D), 1 + 0.1 * rand(D)
    freq, amplitude = gpu.rope_freq(64, 1e7, "yarn", 2.0, 262144)
    freq = freq.cuda()
    pool = torch.zeros(PAGES, 2 * HKV * 64 * 272, dtype=torch.uint8, device="cuda")
    book = PageBook(PAGES)

    def step(seqs, new, group, shared):
        moved = [book.extend(s, n) for s, n in zip(seqs, new)]
        src, dst = [p for m in moved for p in m[0]], [p for m in moved for p in m[1]]
        if src:
            assert gpu.pages_copy(pool, pool.shape[1], PAGES, torch.tensor(src, dtype=torch.int32), torch.tensor(dst, dtype=torch.int32), len(src)) == 0
        n = sum(new)
        proj, k, v = rand(n, H, 2 * D), rand(n, HKV, D), rand(n, HKV, D)
        table, lens = book.tables(seqs)
        view = gpu.Pages(pool, ints(table), ints(lens), ints(starts(new)), 1, HKV, n)
        q = torch.empty(n, H, D, device="cuda")
        assert view.write(0, proj, k, v, wq, wk, None, freq, q, H, 64, 0, amplitude, H * 2 * D, 2 * D, HKV * D, D, HKV * D, D, 1e-6) == 0
        ws = torch.empty(view.attn_shared_workspace(len(shared), H), dtype=torch.uint8, device="cuda")
        out, plain = torch.empty_like(q), torch.empty_like(q)
        assert view.attn_shared(0, ints(group), ints(shared), q, out, H, ws, D ** -0.5) == 0
        size = view.attn_workspace(max(lens), H)
        assert view.attn(0, q, plain, H, max(lens), torch.empty(size, dtype=torch.uint8, device="cuda") if size else None, D ** -0.5) == 0
        assert bool(((out - plain).abs() <= 2e-5 * plain.abs().amax(-1, keepdim=True)).all())
        return view, lens

    prompt = book.new()
    step([prompt], [PROMPT], [0, 1], [0])
    answers = [book.fork(prompt) for _ in range(N)]
    for i in range(70):
        step(answers, [1 if (i + s) % 5 else 2 for s in range(N)], [0, N], [PROMPT // 64])
    # the oldest page of an answer dropped
    s = answers[0]
    table, lens = book.tables([s])
    n = lens[0] - 64
    view = gpu.Pages(pool, ints(table), ints(lens), ints([0, n]), 1, HKV, n)
    k, v, back = (torch.empty(n, HKV, D, device="cuda") for _ in range(3))
    assert view.read(0, ints([64]), k, v) == 0
    none, pos = torch.empty(0, device="cuda"), torch.full((n,), -64, dtype=torch.int32, device="cuda")
    assert gpu.rope(none, k, pos, freq, none, back, n, 0, HKV, D, 64, 0, 1.0, 0, 0, HKV * D, D) == 0
    moved = book.new()
    assert book.extend(moved, n) == ([], [])
    table, lens = book.tables([moved])
    view = gpu.Pages(pool, ints(table), ints(lens), ints([0, n]), 1, HKV, n)
    assert view.append(0, back, v) == 0
    kr, vr = torch.empty_like(k), torch.empty_like(k)
    assert view.read(0, None, kr, vr) == 0
    assert torch.equal(vr, v)                           # codes of codes times a scale: themselves (the largest has code 127)
    # keys: a code more, half a step of a block's largest value over 127 (and 2^-11 of it, the scale's), of what they are at their new positions
    t = (-64 * freq)[None, None]
    want = k.double()
    a, b = want[..., :32].clone(), want[..., 32:64].clone()
    want[..., :32], want[..., 32:64] = a * t.cos() - b * t.sin(), b * t.cos() + a * t.sin()
    most = want.reshape(n, HKV, 8, 32).abs().amax(-1, keepdim=True)
    assert bool(((kr.double() - want).reshape(n, HKV, 8, 32).abs() <= most * (0.5 / 127 + 2 ** -11) * 1.001).all())
    step([moved], [3], [0, 1], [0])
