"""Rotary positions and the calls around shared pages: what is refused before anything is launched, tables of frequencies, workspace sizes."""
import ctypes as C
import math

import pytest

from test_sequences_cpu import BAD_CACHES, ONE, struct


def test_rope_refusals():
    import bonsai_b200
    f = bonsai_b200.lib().bonsai_b200_rope

    def call(n_tok=2, n_head=4, n_head_kv=2, dim=256, n_rot=64, pairs=0, amplitude=1.0, qt=1024, qh=256, kt=512, kh=256, q=ONE, k=32, pos=ONE, freq=ONE, q_out=64, k_out=80):
        return f(q, k, pos, freq, q_out, k_out, n_tok, n_head, n_head_kv, dim, n_rot, pairs, amplitude, qt, qh, kt, kh, None)
    for bad in ({"dim": 0}, {"dim": 257}, {"n_rot": 63}, {"n_rot": 258}, {"n_rot": -2}, {"n_head": -1}, {"n_head_kv": -1}, {"q": None}, {"q": 18}, {"k": None}, {"pos": None}, {"pos": 18},
                {"freq": None}, {"freq": 20}, {"pairs": 2}, {"pairs": -1}, {"amplitude": math.inf}, {"amplitude": math.nan}, {"qh": 255}, {"qt": 1023}, {"qt": -1024}, {"kt": 511},
                {"n_tok": 1 << 31}, {"q_out": None}, {"q_out": 66}, {"k_out": None}, {"qt": 0, "qh": 512}, {"qt": 100, "qh": 512}, {"qt": 1 << 61, "qh": 1 << 44},
                {"q_out": 32}, {"k_out": ONE},          # an output in the place of the other input
                {"q_out": ONE, "qt": 2048}, {"k_out": 32, "kt": 1024}, {"q_out": ONE, "qt": 256, "qh": 512}):       # in the place of an input that is not packed
        assert call(**bad) == 1, bad
    assert call(n_tok=0) == 0 and call(n_head=0, n_head_kv=0) == 0 and call(n_tok=-1) == 0


def test_frequencies():
    import bonsai_b200 as bb
    for n_rot, theta, factor, trained in ((64, 1e7, 1.0, 262144), (64, 1e7, 4.0, 262144), (128, 1e4, 8.0, 4096), (256, 5e5, 32.0, 8192), (6, 100.0, 3.0, 50), (4, 1e4, 2.0, 1)):
        plain = [theta ** (-2.0 * i / n_rot) for i in range(n_rot // 2)]

        def got(kind):
            freq, amplitude = bb.rope_freq(n_rot, theta, kind, factor, trained)
            return freq.tolist(), amplitude
        same = lambda a, b: all(abs(x - y) <= 1e-13 * y for x, y in zip(a, b, strict=True))  # noqa: E731
        f, a = got("plain")
        assert same(f, plain) and a == 1.0
        f, a = got("linear")
        assert same(f, [x / factor for x in plain]) and a == 1.0
        f, a = got("base")
        assert a == 1.0 and f[0] == 1.0 and abs(f[-1] * factor / plain[-1] - 1) < 1e-12
        assert same(f, [(theta * factor ** (n_rot / (n_rot - 2))) ** (-2.0 * i / n_rot) for i in range(n_rot // 2)])
        f, a = got("yarn")
        assert abs(a - (0.1 * math.log(factor) + 1)) <= 2 ** -24 * a
        if factor == 1.0:
            assert same(f, plain)
        # the pair that turns r times in the trained positions: theta^(-2 i / n_rot) trained = 2 pi r
        number = lambda r: n_rot * math.log(trained / (r * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(0, math.floor(number(32))), min(n_rot - 1, math.ceil(number(1)))
        for i, (x, y) in enumerate(zip(f, plain)):
            if i <= low and high > low:
                assert abs(x - y) <= 1e-13 * y
            elif i >= high:
                assert abs(x - y / factor) <= 1e-13 * y
            else:
                part = (i - low) / (high - low)
                assert abs(x - (y * (1 - part) + y / factor * part)) <= 1e-13 * y


def test_frequencies_that_are_refused():
    import bonsai_b200 as bb
    for bad in ((0, 1e4), (-2, 1e4), (63, 1e4), (64, 1.0), (64, 0.5), (64, math.inf), (64, math.nan), (64, 1e4, "linear", 0.5), (64, 1e4, "linear", math.nan), (64, 1e4, "linear", math.inf),
                (64, 1e4, "yarn", 2.0, 0), (64, 1e4, "yarn", 2.0, -1), (2, 1e4, "base", 2.0)):
        with pytest.raises(RuntimeError):
            bb.rope_freq(*bad)
    with pytest.raises(KeyError):
        bb.rope_freq(64, 1e4, "other")
    f, a = (C.c_double * 32)(), C.c_float()
    L = bb.lib()
    for kind in (-1, 4):
        assert L.bonsai_b200_rope_freq(f, C.byref(a), 64, 1e4, kind, 1.0, 0) == 1
    assert L.bonsai_b200_rope_freq(None, C.byref(a), 64, 1e4, 0, 1.0, 0) == 1 and L.bonsai_b200_rope_freq(f, None, 64, 1e4, 0, 1.0, 0) == 1


def test_write_and_read_refusals():
    import bonsai_b200
    L = bonsai_b200.lib()

    def write(layer=0, q=16, k=32, v=48, wq=64, wk=64, pos=None, freq=ONE, out=80, n_head=24, n_rot=64, pairs=0, amplitude=1.0, qt=6144, qh=256, kt=1024, kh=256, vt=1024, vh=256, **kw):
        return L.bonsai_b200_pages_write(C.byref(struct(**kw)), layer, q, k, v, wq, wk, pos, freq, out, n_head, n_rot, pairs, amplitude, qt, qh, kt, kh, vt, vh, 1e-6, None)

    def read(layer=0, first=None, k=ONE, v=32, kind=0, **kw):
        return L.bonsai_b200_pages_read(C.byref(struct(**kw)), layer, first, k, v, kind, None)
    for bad in BAD_CACHES + ({"layer": -1}, {"layer": 2}):
        assert write(**bad) == 1, bad
        assert read(**bad) == 1, bad
    for bad in ({"q": None}, {"q": 18}, {"k": None}, {"v": None}, {"v": 50}, {"wq": 66}, {"wk": 66}, {"pos": 18}, {"freq": None}, {"freq": 20}, {"out": None}, {"out": 82}, {"n_head": -1},
                {"n_rot": 258}, {"n_rot": 3}, {"pairs": 2}, {"amplitude": math.nan}, {"qt": 6143}, {"qh": 255}, {"kt": 1023}, {"vt": 1023}, {"vh": 0}, {"out": 32}, {"out": 48},
                {"out": 16, "qt": 12288, "qh": 512}):
        assert write(**bad) == 1, bad
    for bad in ({"k": None, "v": None}, {"k": 32}, {"k": 24}, {"v": 40}, {"first": 18}, {"kind": 3}, {"kind": -1}):
        assert read(**bad) == 1, bad
    for none in ({"n_seq": 0}, {"n_tok": 0}):
        assert write(**none) == 0 and read(**none) == 0


def test_attention_refusals():
    import bonsai_b200
    L = bonsai_b200.lib()
    need = L.bonsai_b200_pages_attn_shared_workspace(C.byref(struct()), 1, 24)
    assert need > 0

    def attn(layer=0, group=ONE, shared=ONE, n_groups=1, q=ONE, out=32, n_head=24, ws=ONE, ws_bytes=need, **kw):
        return L.bonsai_b200_pages_attn_shared(C.byref(struct(**kw)), layer, group, shared, n_groups, q, out, n_head, ws, ws_bytes, 0.0625, None)
    for bad in BAD_CACHES + ({"layer": -1}, {"layer": 2}, {"group": None}, {"shared": None}, {"group": 18}, {"shared": 18}, {"n_groups": -1}, {"n_groups": 3}, {"q": None}, {"q": 18}, {"out": None},
                             {"out": 34}, {"n_head": 0}, {"n_head": -4}, {"n_head": 6}, {"ws": None}, {"ws": 24}, {"ws_bytes": need - 1}, {"table_stride": (1 << 24) + 1}):
        assert attn(**bad) == 1, bad
    assert attn(n_seq=0, n_groups=0) == 0 and attn(n_tok=0) == 0
    assert L.bonsai_b200_pages_attn_shared(None, 0, None, None, 0, ONE, ONE, 24, ONE, need, 0.0625, None) == 1


@pytest.mark.parametrize("n_head,n_head_kv", [(24, 4), (6, 6), (32, 1), (64, 64), (5, 1)])
def test_workspaces(n_head, n_head_kv):
    """Parts: each row of a call twice, and a tile of 48 rows (128 of images) for each of 148 CTAs.  Images: of calls of more than 640 rows, 2.5 GB at most."""
    import bonsai_b200
    size = bonsai_b200.lib().bonsai_b200_pages_attn_shared_workspace

    def bytes_of(groups=1, head=n_head, **kw):
        p = struct(**{"n_head_kv": n_head_kv, **kw})
        return size(C.byref(p), groups, head)
    row, group, most = 4 * 256 + 8, n_head // n_head_kv, 0
    for n_tok in (1, 7, 640 // group, 640 // group + 1, 5000):
        for n_pages in (1, 100, 100000):
            for stride in (1, 500):
                got = bytes_of(n_tok=n_tok, n_pages=n_pages, table_stride=stride)
                parts = (2 * n_tok * n_head + 148 * 48) * row
                image = 0
                if n_tok * group > 640:
                    parts += 148 * 128 * row
                    image = min(n_pages, 2 * n_tok * group // 641 * stride) * n_head_kv * 133 * 1024
                assert parts <= got <= parts + min(image, int(2.5 * 2 ** 30)) + 16384 and got % 16 == 0, (n_tok, n_pages, stride)
                most = max(most, got - parts)
    assert most <= 2.5 * 2 ** 30 + 16384
    for bad in ({"groups": 3}, {"groups": -1}, {"head": 0}, {"n_tok": 0}, {"n_seq": 0}, {"n_pages": 0}, {"table_stride": 0}, {"n_head_kv": 0}, {"n_head_kv": 1 << 17}, {"n_tok": 1 << 30, "head": 64 * n_head_kv}):
        assert bytes_of(**bad) == 0, bad
    assert bonsai_b200.lib().bonsai_b200_pages_attn_shared_workspace(None, 0, 24) == 0
    if n_head_kv > 1:
        assert bytes_of(head=n_head + 1) == 0


def test_python_refusals():
    """Arguments are looked at before the library is called."""
    import bonsai_b200 as bb
    import torch
    x, f = torch.zeros(4096), torch.zeros(32, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        bb.rope(x, x, torch.zeros(2, dtype=torch.int32), f, x, x, 2, 4, 2, 64, 64, 0, 1.0, 256, 64, 128, 64)
