"""Calls for several sequences: what is refused before anything is launched, workspace sizes, and the host's book of pages."""
import ctypes as C
import random

import pytest

ONE = 16            # an aligned address that no refused call reads


def test_head_norm_refusals():
    import bonsai_b200
    f = bonsai_b200.lib().bonsai_b200_qk_norm_rope

    def call(n_tok=2, n_head=4, n_head_kv=2, dim=256, n_rot=64, qt=1024, qh=256, kt=512, kh=256, q=ONE, pos=ONE, freq=ONE):
        return f(q, ONE, ONE, ONE, pos, freq, ONE, ONE, n_tok, n_head, n_head_kv, dim, n_rot, qt, qh, kt, kh, 1e-6, None)
    for bad in ({"dim": 0}, {"dim": 257}, {"n_rot": 63}, {"n_rot": 258}, {"n_rot": -2}, {"n_head": -1}, {"n_head_kv": -1}, {"q": None}, {"q": 18}, {"pos": None},
                {"freq": None}, {"freq": 20}, {"qh": 255}, {"qt": 1023}, {"qt": -1024}, {"kt": 511}, {"n_tok": 1 << 31}):
        assert call(**bad) == 1, bad
    assert call(n_tok=0) == 0 and call(n_head=0, n_head_kv=0) == 0


def test_head_norm_rows_that_overlap():
    """Tokens that lie closer than a row, whichever of the strides is the larger one."""
    import bonsai_b200
    f = bonsai_b200.lib().bonsai_b200_qk_norm_rope

    def call(n_tok, n_head, qt, qh, n_head_kv=0, kt=0, kh=0):
        return f(ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, n_tok, n_head, n_head_kv, 256, 64, qt, qh, kt, kh, 1e-6, None)
    for qt, qh in ((0, 512), (100, 512), (255, 1024), (255, 1 << 40)):
        assert call(2, 4, qt, qh) == 1, (qt, qh)
        assert call(2, 0, 0, 0, 4, qt, qh) == 1, (qt, qh)
    assert call(3, 4, 300, 512) == 1 and call(2, 4, 512, 300) == 1             # rows of one token in front of another's
    assert call(1 << 20, 4, 1 << 61, 1 << 44) == 1                             # spans past 64 bits
    assert call(2, 1, 255, 0) == 1


def test_head_norm_outputs_in_the_place_of_inputs():
    """Only row for row: where the input is packed."""
    import bonsai_b200
    f = bonsai_b200.lib().bonsai_b200_qk_norm_rope

    def call(q_out, k_out, n_tok=2, qt=1024, qh=256, n_head_kv=2, kt=512, kh=256):
        return f(16, 32, ONE, ONE, ONE, ONE, q_out, k_out, n_tok, 4, n_head_kv, 256, 64, qt, qh, kt, kh, 1e-6, None)
    assert call(16, 64, qt=2048, qh=512) == 1 and call(64, 32, kt=1024) == 1 and call(16, 64, n_tok=1, qh=512) == 1
    assert call(16, 64, qt=256, qh=512) == 1            # heads first, then tokens
    assert call(32, 64) == 1 and call(64, 16) == 1      # the other input


def struct(**kw):
    import bonsai_b200
    have = dict(pool=ONE, table=ONE, len=ONE, start=ONE, n_pages=4, n_layers=2, n_head_kv=4, n_seq=2, table_stride=3, n_tok=5)
    have.update(kw)
    return bonsai_b200.PagesStruct(**have)


BAD_CACHES = ({"pool": None}, {"pool": 24}, {"table": None}, {"table": 18}, {"len": None}, {"start": 17}, {"n_pages": 0}, {"n_layers": 0}, {"n_head_kv": 0}, {"n_seq": -1},
              {"table_stride": 0}, {"n_tok": -1})


def test_cache_refusals():
    import bonsai_b200
    L = bonsai_b200.lib()

    def append(layer=0, k=ONE, v=ONE, **kw):
        return L.bonsai_b200_pages_append(C.byref(struct(**kw)), layer, k, v, None)

    def attn(layer=0, q=ONE, out=ONE, n_head=24, max_len=100, ws=None, ws_bytes=0, **kw):
        return L.bonsai_b200_pages_attn(C.byref(struct(**kw)), layer, q, out, n_head, max_len, ws, ws_bytes, 0.0625, None)
    for bad in BAD_CACHES + ({"layer": -1}, {"layer": 2}):
        assert append(**bad) == 1, bad
        assert attn(**bad) == 1, bad
    assert append(k=None) == 1 and append(v=18) == 1
    assert L.bonsai_b200_pages_append(None, 0, ONE, ONE, None) == 1
    assert attn(n_head=0) == 1 and attn(n_head=6) == 1 and attn(max_len=-1) == 1 and attn(q=None) == 1 and attn(out=18) == 1
    for none in ({"n_seq": 0}, {"n_tok": 0}):
        assert append(**none) == 0 and attn(**none) == 0
    # a workspace that is too small, missing or not aligned
    need = L.bonsai_b200_pages_attn_workspace(5, 30000, 2, 24, 4)
    assert need > 0
    assert attn(max_len=30000) == 1 and attn(max_len=30000, ws=ONE, ws_bytes=need - 1) == 1 and attn(max_len=30000, ws=24, ws_bytes=need) == 1


def test_tables_of_too_many_positions():
    """Positions are counted in 32 bits: a table row has room for 2^30 of them at most."""
    import bonsai_b200
    L = bonsai_b200.lib()
    for stride in ((1 << 24) + 1, 1 << 25, (1 << 31) - 1):
        p = struct(table_stride=stride)
        assert L.bonsai_b200_pages_append(C.byref(p), 0, ONE, ONE, None) == 1
        assert L.bonsai_b200_pages_attn(C.byref(p), 0, ONE, ONE, 24, 1, None, 0, 0.0625, None) == 1
    need = L.bonsai_b200_pages_attn_workspace(5, (1 << 31) - 1, 2, 24, 4)
    assert 0 < need < 1 << 30


def test_workspace_sizes():
    import bonsai_b200 as bb
    assert bb.pages_attn_workspace(1, 64, 1, 24, 4) == 0
    for bad in ((0, 64, 1, 24, 4), (1, 0, 1, 24, 4), (1, 64, 0, 24, 4), (1, 64, 1, 24, 5), (1, 64, 1, 0, 4), (1, 64, 1, 24, 0), (1 << 30, 64, 1, 24, 4)):
        assert bb.pages_attn_workspace(*bad) == 0
    assert bb.pages_attn_workspace(1, 262144, 1, 24, 4) % 16 == 0
    for bad in ((0, 1, 16, 48, 128, 128), (1, 0, 16, 48, 128, 128), (1, 1, 16, 47, 128, 128), (1, 1, 16, 48, 129, 128), (1, 1, 16, 48, 128, 100)):
        assert bb.gdn_seqs_workspace(*bad) == 0


@pytest.mark.parametrize("n_head,n_head_kv", [(24, 4), (6, 6), (32, 1), (64, 64), (5, 1)])
def test_workspaces_are_bounded(n_head, n_head_kv):
    """Sums of CTAs that share a tile: at most twice as many tiles as CTAs run at once (2 per SM) of 8 and of 64 rows, and beside prompts 8 tiles of 128 rows per SM.  Images: 2.5 GB."""
    import bonsai_b200 as bb
    row = 4 * 256 + 8
    few, tc = 2 * 2 * 148 * (8 + 64) * row, 8 * 148 * 128 * row
    for n_tok in (1, 5, 33, 128, 512, 800, 2049, 5333, 16384, 100000):
        for max_len in (1, 129, 2501, 20400, 40000, 262144, 1 << 30):
            for n_seq in (1, 2, 16, 17, 1000, 100000):
                size = bb.pages_attn_workspace(n_tok, max_len, n_seq, n_head, n_head_kv)
                assert size <= few + tc + (5 << 29) + (1 << 24), (n_tok, max_len, n_seq, size)
                if n_tok * (n_head // n_head_kv) < 256:         # no prompts
                    assert size <= few + 64
    # many tokens of sequences that may be long, for whose images there is no room
    for n_tok, max_len, n_seq in ((2049, 262144, 2), (2015, 20400, 16), (8192, 40000, 16)):
        assert bb.pages_attn_workspace(n_tok, max_len, n_seq, 24, 4) <= few + 64


def test_copy_refusals():
    import bonsai_b200
    f = bonsai_b200.lib().bonsai_b200_pages_copy

    def call(src, dst, pool=ONE, page_bytes=32, n_pages=8):
        n = len(src)
        ints = lambda v: (C.c_int32 * max(1, n))(*v)  # noqa: E731
        return f(pool, page_bytes, n_pages, ints(src), ints(dst), n, None)
    assert call([0], [8]) == 1 and call([-1], [0]) == 1 and call([8], [0]) == 1 and call([0], [-1]) == 1
    assert call([0, 1], [5, 5]) == 1            # written twice
    assert call([0, 5], [5, 6]) == 1            # written and read, either order
    assert call([5, 0], [6, 5]) == 1
    assert call([3], [3]) == 1
    assert call([0], [1], pool=None) == 1 and call([0], [1], pool=8) == 1 and call([0], [1], page_bytes=24) == 1 and call([0], [1], page_bytes=0) == 1
    assert call([0], [1], n_pages=0) == 1
    assert call([], []) == 0
    assert f(ONE, 32, 8, None, None, 1, None) == 1 and f(ONE, 32, 8, None, None, -1, None) == 1


def test_delta_refusals():
    import bonsai_b200
    f = bonsai_b200.lib().bonsai_b200_gdn_seqs

    def call(state=ONE, start=ONE, slot=None, n_seq=2, n_slots=2, n_tok=5, kh=16, vh=48, K=128, V=128):
        return f(state, ONE, ONE, ONE, ONE, ONE, ONE, start, slot, None, 0, n_seq, n_slots, n_tok, kh, vh, K, V, None)
    for bad in ({"state": None}, {"start": 18}, {"slot": 18}, {"n_seq": -1}, {"n_slots": 1}, {"n_slots": -1, "slot": ONE}, {"n_tok": -1}, {"kh": 15}, {"vh": 0}, {"kh": 0}, {"K": 0},
                {"K": 129}, {"V": 33}, {"V": 0}, {"n_seq": 65536, "n_slots": 65536}):
        assert call(**bad) == 1, bad
    assert call(n_tok=0) == 0 and call(n_seq=0) == 0


def test_python_refusals():
    import torch
    import bonsai_b200 as bb
    x = torch.zeros(64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        bb.qk_norm_rope(x, x, x, x, x, x, x, x, 1, 1, 1, 64, 0, 64, 64, 64, 64, 1e-6)
    with pytest.raises(RuntimeError, match="no CPU path"):
        bb.gdn_seqs(x, x, x, x, x, x, x, x, None, None, 0, 1, 1, 1, 1, 1, 32, 32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        bb.Pages(x.byte(), x.int().reshape(1, -1), x[:1].int(), x[:2].int(), 1, 1, 1)


@pytest.mark.parametrize("exponent", [6, -8, -12, -20])
def test_scales_by_product_and_by_quotient(exponent):
    """Largest magnitude times 1 / 127 and over 127 are the same fp16 scale for every fp32 magnitude (normal ones and subnormal ones), though not the same fp32 scale."""
    import numpy as np
    x = (np.arange(1 << 23, dtype=np.uint32) | np.uint32(127 << 23)).view(np.float32) * np.float32(2.0 ** exponent)

    def half(d):
        d = d.astype(np.float64)
        step = np.ldexp(1.0, np.maximum(np.frexp(d)[1] - 1, -14) - 10)
        return np.floor(d / step + 0.5) * step
    product, quotient = x * (np.float32(1) / np.float32(127)), x / np.float32(127)
    assert 0.04 < (product != quotient).mean() < 0.05
    assert np.array_equal(half(product), half(quotient))


# ---- the book ------------------------------------------------------------------------------------------
def check(book, n_pages):
    users = [0] * n_pages
    for pages, length in book._seqs.values():
        assert len(pages) == -(-length // 64) and len(set(pages)) == len(pages)
        for p in pages:
            users[p] += 1
    assert users == book.users and sorted(book._free) == [p for p in range(n_pages) if not users[p]]


def test_book_against_contents():
    """What each position holds, followed through a thousand random calls by a pool of marks."""
    from bonsai_b200.pages import NoRoom, PageBook
    rng = random.Random(7)
    n_pages = 40
    book, pool, want, mark = PageBook(n_pages), [[None] * 64 for _ in range(n_pages)], {}, 0

    def copy(src, dst):
        assert len(src) == len(dst) and not set(src) & set(dst) and len(set(dst)) == len(dst)
        for s, d in zip(src, dst):
            pool[d] = list(pool[s])
    for _ in range(1000):
        seqs = list(want)
        op = rng.choice(["new", "extend", "extend", "extend", "fork", "truncate", "free", "compact"])
        if op == "new" and len(seqs) < 8:
            want[book.new()] = []
        elif op == "compact":
            copy(*book.compact())
            used = n_pages - book.free_pages
            assert all(book.users[:used]) and not any(book.users[used:])
        elif seqs:
            s = rng.choice(seqs)
            if op == "extend":
                n, was = rng.choice([0, 1, 5, 63, 64, 130]), (list(book.users), book.pages(s), book.length(s))
                try:
                    copy(*book.extend(s, n))
                except NoRoom:
                    assert was == (book.users, book.pages(s), book.length(s))
                    continue
                for _ in range(n):
                    mark += 1
                    p = len(want[s])
                    pool[book.pages(s)[p // 64]][p % 64] = mark
                    want[s].append(mark)
            elif op == "fork" and len(seqs) < 8:
                want[book.fork(s)] = list(want[s])
            elif op == "truncate":
                n = rng.randint(0, len(want[s]))
                book.truncate(s, n)
                del want[s][n:]
            elif op == "free" and rng.random() < 0.3:
                book.free(s)
                del want[s]
        check(book, n_pages)
        for s, marks in want.items():
            assert book.length(s) == len(marks)
            assert [pool[book.pages(s)[p // 64]][p % 64] for p in range(len(marks))] == marks


def test_book_refusals():
    from bonsai_b200.pages import NoRoom, PageBook
    with pytest.raises(ValueError):
        PageBook(0)
    book = PageBook(2)
    s = book.new()
    assert book.extend(s, 65) == ([], [])
    with pytest.raises(NoRoom):
        book.extend(s, 64)
    with pytest.raises(ValueError):
        book.extend(s, -1)
    with pytest.raises(ValueError):
        book.truncate(s, 66)
    with pytest.raises(ValueError):
        book.tables([s], 1)
    assert book.tables([s], 3) == ([[0, 1, 0]], [65])
    t = book.fork(s)
    with pytest.raises(NoRoom):                 # the shared last page would have to be copied
        book.extend(t, 1)
    book.free(s)
    assert book.extend(t, 1) == ([], []) and book.free_pages == 0
    with pytest.raises(KeyError):
        book.length(s)
