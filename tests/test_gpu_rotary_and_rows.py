"""Rotary positions and the rows of a paged cache, written from projections and read back, against plain statements in 64 bits and in rounded steps."""
import math

import numpy as np
import pytest

from test_gpu_sequences import U, Cache, blocks, ints, number, starts, status_is_clear  # noqa: F401

pytestmark = pytest.mark.gpu


def turned(x, pos, freq, n_rot, pairs, amplitude):
    """In 64 bits, and the magnitudes that an output is a sum of."""
    import torch
    y = x.double()
    y, size = y.clone(), y.abs()
    if n_rot:
        h = n_rot // 2
        t = (pos.double()[:, None] * freq)[:, None]
        c, s = t.cos() * amplitude, t.sin() * amplitude
        a, b = (slice(0, n_rot, 2), slice(1, n_rot, 2)) if pairs else (slice(0, h), slice(h, n_rot))
        p, q = y[..., a].clone(), y[..., b].clone()
        y[..., a], y[..., b] = p * c - q * s, q * c + p * s
        size[..., a], size[..., b] = (p * c).abs() + (q * s).abs(), (q * c).abs() + (p * s).abs()
    return y, size


# A sine or cosine is rounded once (and 2^-52 off in 64 bits), each product and their sum once: 3 u and a bit of |a c| + |b s|
ROPE_ROUNDINGS = 3.01
SHAPES = [  # tokens, heads, kv heads, head_dim, n_rot
    (1, 24, 4, 256, 64), (1, 1, 1, 256, 256), (7, 24, 4, 256, 64), (300, 24, 4, 256, 64), (33, 8, 8, 128, 128), (5, 3, 1, 64, 62), (3, 40, 8, 100, 20), (4, 6, 2, 64, 8),
    (2, 5, 2, 33, 0), (9, 2, 1, 2, 2), (4, 6, 3, 254, 2), (17, 0, 4, 256, 64), (17, 24, 0, 256, 64), (1300, 4, 2, 36, 8), (2, 700, 3, 64, 32), (400, 64, 8, 128, 128)]


@pytest.mark.parametrize("n_tok,n_head,n_head_kv,dim,n_rot", SHAPES)
@pytest.mark.parametrize("pairs", [0, 1])
@pytest.mark.parametrize("layout", ["packed", "beside a gate", "odd", "in place", "heads first"])
def test_rope(gpu, n_tok, n_head, n_head_kv, dim, n_rot, pairs, layout):
    import torch
    g = torch.Generator(device="cuda").manual_seed(n_tok * 1000 + dim)
    wide, odd = {"beside a gate": (2 * dim, 0), "odd": (dim + 3, 1)}.get(layout, (dim, 0))

    def rows(heads):
        first, second = (heads, n_tok) if layout == "heads first" else (n_tok, heads)
        x = torch.randn(n_tok * heads * wide + odd, generator=g, device="cuda")[odd:].reshape(first, second, wide)
        x *= torch.exp(4 * torch.randn(first, second, 1, generator=g, device="cuda"))
        return x.transpose(0, 1) if layout == "heads first" else x
    q, k = rows(n_head), rows(n_head_kv)
    pos = torch.randint(0, 262144, (n_tok,), generator=g, device="cuda", dtype=torch.int32)
    pos[0] = 262143
    if n_tok > 3:
        pos[1], pos[2], pos[3] = 0, -64, 2 ** 31 - 1
    freq, amplitude = gpu.rope_freq(max(n_rot, 4), 1e7, "yarn", 4.0, 262144)
    freq, amplitude = freq[:n_rot // 2].cuda(), float(np.float32(amplitude))
    wants = [turned(x[..., :dim], pos, freq, n_rot, pairs, amplitude) for x in (q, k)]
    empty = lambda h: torch.full((n_tok * h * dim + odd + 8,), 7.0, device="cuda")[odd:]  # noqa: E731
    outs = [q, k] if layout == "in place" else [empty(n_head), empty(n_head_kv)]
    strides = [s for x, heads in ((q, n_head), (k, n_head_kv)) for s in ((wide, n_tok * wide) if layout == "heads first" else (heads * wide, wide))]
    assert gpu.rope(q, k, pos, freq, *outs, n_tok, n_head, n_head_kv, dim, n_rot, pairs, amplitude, *strides) == 0
    for out, (want, size), heads in zip(outs, wants, (n_head, n_head_kv)):
        n = n_tok * heads * dim
        got = out.reshape(-1)[:n].reshape(want.shape)
        assert bool(((got.double() - want).abs() <= ROPE_ROUNDINGS * U * size).all())
        assert torch.equal(got[..., n_rot:].double(), want[..., n_rot:])
        assert layout == "in place" or bool((out[n:] == 7).all())


def test_rope_of_odd_values(gpu):
    """An infinity or NaN stays in its pair; positions all over, there and back."""
    import torch
    x = torch.randn(3, 2, 64, device="cuda")
    x[1, 1, 3], x[2, 0, 5] = math.inf, math.nan
    none = torch.empty(0, device="cuda")
    freq = torch.ones(16, dtype=torch.float64, device="cuda")
    for pairs, partners in ((0, (19, 21)), (1, (2, 4))):
        out = torch.empty_like(x)
        assert gpu.rope(x, none, ints([1, 2, 3]), freq, out, none, 3, 2, 0, 64, 32, pairs, 1.0, 128, 64, 0, 0) == 0
        bad = torch.zeros(3, 2, 64, dtype=torch.bool, device="cuda")
        bad[1, 1, [3, partners[0]]], bad[2, 0, [5, partners[1]]] = True, True
        assert torch.equal(~out.isfinite(), bad)
    x = torch.randn(50, 2, 64, device="cuda")
    there, back = torch.empty_like(x), torch.empty_like(x)
    pos = torch.arange(50, dtype=torch.int32, device="cuda") * 5000
    call = lambda a, p, b: gpu.rope(a, none, p, freq, b, none, 50, 2, 0, 64, 32, 0, 1.0, 128, 64, 0, 0)  # noqa: E731
    assert call(x, pos, there) == 0 and call(there, -pos, back) == 0
    most = x.abs().amax(-1, keepdim=True).double()
    assert bool(((back - x).abs() <= 2 * 2 * 2 * ROPE_ROUNDINGS * U * most).all())              # two turns, sums of two, turned on by sine and cosine


# ---- rows written ----------------------------------------------------------------------------------------
def plain_rows(x, w, pos, freq, n_rot, pairs, amplitude, eps):
    """Norm and rotation of [tokens][heads][256] in the roundings that are stated (numpy)."""
    f32 = np.float32
    x = x.astype(f32)
    if w is not None:
        scale = (1 / np.sqrt((x.astype(np.float64) ** 2).sum(-1, keepdims=True) / 256 + np.float64(f32(eps)))).astype(f32)
        x = (x * scale).astype(f32) * w
    if n_rot:
        t = (pos.astype(np.float64)[:, None] * freq)[:, None]
        c, s = (np.cos(t) * np.float64(f32(amplitude))).astype(f32), (np.sin(t) * np.float64(f32(amplitude))).astype(f32)
        a, b = (slice(0, n_rot, 2), slice(1, n_rot, 2)) if pairs else (slice(0, n_rot // 2), slice(n_rot // 2, n_rot))
        p, q = x[..., a].copy(), x[..., b].copy()
        x = x.copy()
        x[..., a], x[..., b] = p * c - q * s, q * c + p * s
    return x


ROWS = [  # lengths, new tokens, query heads, kv heads, rows of nobody
    ([1], [1], 24, 4, 0), ([65], [2], 3, 1, 3), ([200, 3, 64, 0, 129], [70, 3, 1, 0, 0], 24, 4, 2), ([40] * 30, [1] * 30, 8, 2, 0), ([700], [500], 24, 4, 1), ([130], [128], 0, 3, 0),
    ([90], [90], 70, 2, 0), ([1300], [1201], 14, 1, 1), ([1, 64, 65], [1, 1, 1], 5, 5, 0)]


@pytest.mark.parametrize("lens,new,n_head,n_head_kv,behind", ROWS)
@pytest.mark.parametrize("n_rot,pairs,norm", [(64, 0, True), (256, 0, True), (64, 1, True), (62, 0, True), (0, 0, True), (256, 1, False), (64, 0, False), (0, 0, False), (6, 0, False)])
@pytest.mark.parametrize("layout", ["packed", "beside a gate", "odd"])
def test_write(gpu, lens, new, n_head, n_head_kv, behind, n_rot, pairs, norm, layout):
    """Queries to a tolerance of the roundings; the bytes of the new rows; every other byte as it was."""
    import torch
    c = Cache(gpu, lens, new, n_layers=2, n_head_kv=n_head_kv, behind=behind, seed=len(lens))
    rng = np.random.default_rng(n_rot + n_head)
    wide, odd = {"beside a gate": (512, 0), "odd": (257, 1)}.get(layout, (256, 0))
    eps, amplitude = 1e-6, 1.25

    def rows(heads):
        x = rng.standard_normal((c.n_tok, heads, wide)).astype(np.float32) * np.exp(2 * rng.standard_normal((c.n_tok, heads, 1))).astype(np.float32)
        return x, torch.cat([torch.zeros(odd), torch.from_numpy(x).flatten()]).cuda()[odd:]
    (q, dq), (k, dk), (v, dv) = (rows(h) for h in (n_head, n_head_kv, n_head_kv))
    wq, wk = ((1 + 0.3 * rng.standard_normal(256)).astype(np.float32) if norm else None for _ in range(2))
    weight = lambda w: None if w is None else torch.cat([torch.zeros(odd), torch.from_numpy(w)]).cuda()[odd:]  # noqa: E731
    freq = 1e7 ** (-np.arange(n_rot // 2) / max(1, n_rot // 2))
    own = np.zeros(c.n_tok, np.int32)
    for s, n in enumerate(new):
        own[c.start[s]:c.start[s] + n] = np.arange(lens[s] - n, lens[s])
    pos = rng.integers(0, 200000, c.n_tok).astype(np.int32) if len(lens) == 1 else None          # said, or where the rows lie
    out = torch.full((c.n_tok * n_head * 256 + odd + 4,), 7.0, device="cuda")[odd:]
    assert c.view.write(1, dq, dk, dv, weight(wq), weight(wk), None if pos is None else ints(pos), torch.from_numpy(freq).cuda(), out, n_head, n_rot, pairs, amplitude, n_head * wide, wide,
                        n_head_kv * wide, wide, n_head_kv * wide, wide, eps) == 0
    mine = sum(new)
    at = own if pos is None else pos
    got = out[:mine * n_head * 256].reshape(mine, n_head, 256).cpu().numpy()
    x = torch.from_numpy(q[:mine, :, :256]).double()
    factor = 1.0
    if norm:                                            # root and product, the weight's: 2.5 u and a bit
        x, factor = x / torch.sqrt((x * x).mean(-1, keepdim=True) + np.float64(np.float32(eps))) * torch.from_numpy(wq).double(), 2.0
    want, size = turned(x, torch.from_numpy(at[:mine]), torch.from_numpy(freq), n_rot, pairs, amplitude)
    assert bool((np.abs(got - want.numpy()) <= (ROPE_ROUNDINGS * factor) * U * size.numpy()).all())
    assert bool((out[mine * n_head * 256:] == 7).all())
    turned_k = plain_rows(k[..., :256], wk, at, freq, n_rot, pairs, amplitude, eps)
    want = c.pool.copy()
    for s, n in enumerate(new):
        for t in range(n):
            p, row = lens[s] - n + t, c.start[s] + t
            want[c.table[s, p // 64], 1, 0, :, p % 64], want[c.table[s, p // 64], 1, 1, :, p % 64] = blocks(turned_k[row]), blocks(v[row, :, :256])
    assert np.array_equal(c.d_pool.cpu().numpy(), want)


@pytest.mark.parametrize("pairs", [0, 1])
def test_write_is_rope_and_append(gpu, pairs):
    """Bit for bit, without norms; queries in the place of the projection."""
    import torch
    a, b = (Cache(gpu, [300, 70], [200, 3], seed=4) for _ in range(2))
    q, k, v = (torch.randn(203, h, 256, device="cuda") for h in (24, 4, 4))
    freq, amplitude = gpu.rope_freq(64, 1e7, "yarn", 4.0, 262144)
    freq = freq.cuda()
    pos = torch.cat([torch.arange(100, 300), torch.arange(67, 70)]).int().cuda()
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    assert gpu.rope(q, k, pos, freq, q_out, k_out, 203, 24, 4, 256, 64, pairs, amplitude, 6144, 256, 1024, 256) == 0
    assert a.view.append(0, k_out, v) == 0
    assert b.view.write(0, q, k, v, None, None, None, freq, q, 24, 64, pairs, amplitude, 6144, 256, 1024, 256, 1024, 256, 1e-6) == 0
    assert torch.equal(q, q_out) and torch.equal(a.d_pool, b.d_pool)


def test_write_of_odd_values(gpu):
    """Zeros, subnormal scales, scales past fp16's largest, infinities and NaN: the bytes that append stores."""
    import torch
    a, b = (Cache(gpu, [100], [6], seed=6) for _ in range(2))
    k, v = torch.randn(6, 4, 256, device="cuda"), torch.randn(6, 4, 256, device="cuda")
    for x in (k, v):
        x[0, 0, :32], x[0, 0, 32:64], x[1, 1, 70], x[2, 2, 100], x[3, 3, 200], x[4, 0] = 0.0, 1e-7, 1e7, math.inf, math.nan, 0.0
    none = torch.empty(0, device="cuda")
    assert a.view.append(0, k, v) == 0
    assert b.view.write(0, none, k, v, None, None, None, None, none, 0, 0, 0, 1.0, 0, 0, 1024, 256, 1024, 256, 1e-6) == 0
    assert torch.equal(a.d_pool, b.d_pool)


# ---- rows read -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("lens,new,first,n_head_kv,behind", [
    ([1], [1], None, 4, 0), ([65], [2], [0], 1, 3), ([200, 3, 64, 0, 129], [70, 3, 1, 0, 0], None, 4, 2), ([500] * 7, [1, 0, 64, 65, 3, 128, 500], [499, 0, 63, 64, 62, 1, 0], 3, 0),
    ([3000, 40], [2500, 1], [17, 39], 8, 1)])
@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("outs", ["kv", "k", "v"])
def test_read(gpu, lens, new, first, n_head_kv, behind, kind, outs):
    import torch
    kind = getattr(torch, kind)
    c = Cache(gpu, lens, new, n_layers=2, n_head_kv=n_head_kv, behind=behind, seed=sum(lens), scale=40.0)
    shape = (c.n_tok, n_head_kv, 256)
    got = [torch.full((c.n_tok + 1, n_head_kv, 256), 7.0, dtype=kind, device="cuda") if x in outs else None for x in "kv"]
    assert c.view.read(1, None if first is None else ints(first), *got) == 0
    for i, x in enumerate(got):
        if x is None:
            continue
        want = np.full((shape[0] + 1, *shape[1:]), 7.0)
        for s, n in enumerate(new):
            at = (lens[s] - n) if first is None else first[s]
            for j in range(n_head_kv):
                want[c.start[s]:c.start[s] + n, j] = c.rows(s, 1, i, j)[at:at + n]
        exact = torch.from_numpy(want).cuda()
        assert torch.equal(exact.float().double(), exact) and torch.equal(x, exact.float().to(kind))


def test_read_of_odd_scales(gpu):
    """Scales that are infinite, no number, subnormal; products beyond fp16."""
    import torch
    c = Cache(gpu, [64], [64], n_head_kv=1)
    flat = c.pool[c.table[0, 0], 0, 0, 0].reshape(64, 8, 34)
    for row, bits in enumerate((0x7C00, 0xFC00, 0x7E00, 0x0001, 0x0000, 0x7BFF, 0x03FF)):
        flat[row, :, :2] = np.array([bits], np.uint16).view(np.uint8)
    c.upload()
    want = torch.from_numpy(number(flat)).float().cuda()
    for kind in (torch.float32, torch.float16, torch.bfloat16):
        k, v = (torch.empty(64, 1, 256, dtype=kind, device="cuda") for _ in range(2))
        assert c.view.read(0, None, k, v) == 0
        assert bool(((k[:, 0] == want.to(kind)) | (k[:, 0].isnan() & want.isnan())).all())


def test_numbers_that_do_not_fit(gpu):
    """Positions and pages that a sequence does not have: the status word says so, the others are served, no other byte changes."""
    import torch
    c = Cache(gpu, [300, 200, 150], [3, 4, 5], seed=10)
    q, k, v = (torch.randn(12, h, 256, device="cuda") for h in (24, 4, 4))
    table, length, start = c.view._keep[1:]

    def write():
        c.d_pool.copy_(torch.from_numpy(c.pool))
        out = torch.full_like(q, 7.0)
        assert c.view.write(0, q, k, v, None, None, None, None, out, 24, 0, 0, 1.0, 6144, 256, 1024, 256, 1024, 256, 1e-6) == 0
        return out, c.d_pool.clone()

    def read(first=None):
        out = [torch.full((12, 4, 256), 7.0, device="cuda") for _ in range(2)]
        assert c.view.read(0, first, *out) == 0
        return out
    (out, pool), rows = write(), read()
    assert torch.equal(out, q) and gpu.device_status() == 0
    others = torch.ones(c.n_pages, dtype=torch.bool, device="cuda")
    others[ints(c.table[1, :4]).long()] = False

    def check():
        assert gpu.device_status() == 0
        o, p = write()
        assert gpu.device_status() == 3 and gpu.clear_status() == 0
        assert torch.equal(o[:3], q[:3]) and torch.equal(o[7:], q[7:]) and bool((o[3:7] == 7).all())
        assert torch.equal(p[others], pool[others]) and torch.equal(p[~others], torch.from_numpy(c.pool).cuda()[~others])
        c.d_pool.copy_(pool)
        for x, want in zip(read(), rows):
            assert gpu.device_status() == 3
            assert torch.equal(x[:3], want[:3]) and torch.equal(x[7:], want[7:]) and bool((x[3:7] == 7).all())
        assert gpu.clear_status() == 0
    for page in (-1, c.n_pages, 2 ** 31 - 1, -2 ** 31):
        table[1, 3] = page
        check()
    table.copy_(ints(c.table))
    for n in (7 * 64, 2 ** 31 - 1):
        length[1] = n
        check()
    length[1] = 200
    for first in ([0, 197, 0], [0, -1, 0], [0, 2 ** 31 - 1, 0], [0, -2 ** 31, 0]):             # partly, or all, behind or in front
        x = read(ints(first))
        assert gpu.device_status() == 3 and gpu.clear_status() == 0
        inside = [t for t in range(4) if 0 <= first[1] + t < 200]
        want = torch.full((4, 4, 256), 7.0, device="cuda")
        for t in inside:
            for j in range(4):
                want[t, j] = torch.from_numpy(number(pool.cpu().numpy()[c.table[1, (first[1] + t) // 64], 0, 0, j, (first[1] + t) % 64].reshape(8, 34))).cuda()
        assert torch.equal(x[0][3:7], want)
    start.copy_(ints([0, 5, 3, 12]))                    # rows that run backwards
    write()
    assert gpu.device_status() == 3 and gpu.clear_status() == 0
    read()
    assert gpu.device_status() == 3 and gpu.clear_status() == 0


def test_tokens_without_a_position(gpu):
    """More new tokens than a sequence has positions: the first ones have no place."""
    import torch
    c = Cache(gpu, [2, 40], [5, 2], seed=3)
    q, k, v = (torch.randn(7, h, 256, device="cuda") for h in (4, 4, 4))
    out = torch.full_like(q, 7.0)
    assert c.view.write(0, q, k, v, None, None, None, None, out, 4, 0, 0, 1.0, 1024, 256, 1024, 256, 1024, 256, 1e-6) == 0
    assert gpu.device_status() == 3 and gpu.clear_status() == 0
    assert bool((out[:3] == 7).all()) and torch.equal(out[3:], q[3:])
    want = c.pool.copy()
    for row, (s, p) in {3: (0, 0), 4: (0, 1), 5: (1, 38), 6: (1, 39)}.items():
        want[c.table[s, 0], 0, 0, :, p], want[c.table[s, 0], 0, 1, :, p] = blocks(k[row].cpu().numpy()), blocks(v[row].cpu().numpy())
    assert np.array_equal(c.d_pool.cpu().numpy(), want)


def test_captured_rows_follow_the_numbers(gpu):
    """Written, read and turned in a captured step, replayed with other lengths and rows; the step by itself on another stream."""
    import torch
    c = Cache(gpu, [700, 300], [200, 3], seed=11, spare=20)
    n = c.n_tok
    q, k, v = (torch.randn(n, h, 256, device="cuda") for h in (24, 4, 4))
    w = torch.rand(256, device="cuda")
    freq = gpu.rope_freq(64, 1e7)[0].cuda()
    out, kr, vr, back, pos = torch.empty_like(q), torch.empty_like(k), torch.empty_like(k), torch.empty_like(k), torch.full((n,), -64, dtype=torch.int32, device="cuda")
    none = torch.empty(0, device="cuda")

    def step():
        return (c.view.write(0, q, k, v, w, w, None, freq, out, 24, 64, 0, 1.0, 6144, 256, 1024, 256, 1024, 256, 1e-6) or c.view.read(0, None, kr, vr) or
                gpu.rope(none, kr, pos, freq, none, back, n, 0, 4, 256, 64, 0, 1.0, 0, 0, 1024, 256))
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(st):
        assert step() == 0
        with torch.cuda.graph(graph, stream=st):
            assert step() == 0
    torch.cuda.synchronize()
    length, start = c.view._keep[2:]
    for lens, new in (([704, 301], [4, 1]), ([640, 64], [0, 64]), ([203, 1], [202, 1])):
        length.copy_(ints(lens))
        start.copy_(ints(starts(new)))
        got = []
        for run in (graph.replay, step):
            c.d_pool.copy_(torch.from_numpy(c.pool))
            for x in (out, kr, vr, back):
                x.fill_(7.0)
            run()
            torch.cuda.synchronize()
            got.append([x.clone() for x in (out, kr, vr, back, c.d_pool)])
        assert all(torch.equal(a, b) for a, b in zip(*got))
        assert bool((got[0][0][sum(new):] == 7).all()) and bool((got[0][1][sum(new):] == 7).all())


def test_what_python_refuses(gpu, monkeypatch):
    import torch
    c = Cache(gpu, [70, 20], [2, 2], seed=17)
    k = torch.empty(4, 4, 256, device="cuda")
    with pytest.raises(RuntimeError, match="of one type"):
        c.view.read(0, None, k, k.half())
    for bad in ((None, None), (k.double(), None), (None, k.int())):
        with pytest.raises(RuntimeError):
            c.view.read(0, None, *bad)
    with pytest.raises(RuntimeError, match="rows of"):
        c.view.read(0, None, k[:3], None)
    with pytest.raises(RuntimeError, match="on device"):
        c.view.read(0, None, k.cpu(), None)
    assert c.view.read(0, None, k, k) == 1              # K and V to one place
    q, freq = torch.empty(4, 24, 256, device="cuda"), torch.ones(32, dtype=torch.float64, device="cuda")
    args = dict(q=q, k=k, v=k, q_weight=None, k_weight=None, pos=None, freq=freq, q_out=torch.empty_like(q))

    def write(**bad):
        a = {**args, **bad}
        return c.view.write(0, *a.values(), 24, 64, 0, 1.0, 6144, 256, 1024, 256, 1024, 256, 1e-6)
    for bad in ({"q": q[:3].clone()}, {"k": k[:3].clone()}, {"v": k[:3].clone()}, {"q_weight": k[0, 0, :255]}, {"k_weight": k[0, 0, :255]}, {"pos": ints([1, 2, 3])}, {"freq": freq[:31]}, {"q_out": q[:3]}, {"freq": freq.float()},
                {"pos": torch.zeros(4, dtype=torch.int64, device="cuda")}, {"k": k.half()}, {"q_out": q.half()}):
        with pytest.raises((RuntimeError, TypeError)):
            write(**bad)
    first = ints([0])
    with pytest.raises((RuntimeError, TypeError)):
        c.view.read(0, first, k, None)
    none = torch.empty(0, device="cuda")
    for bad in ((q[:3].clone(), none, ints([0] * 4), freq, q), (q, none, ints([0] * 3), freq, q), (q, none, ints([0] * 4), freq[:31], q), (q, none, ints([0] * 4), freq, q[:3])):
        with pytest.raises((RuntimeError, TypeError)):
            gpu.rope(*bad, none, 4, 24, 0, 256, 64, 0, 1.0, 6144, 256, 0, 0)
    monkeypatch.setattr(c.view, "_device", c.view._device + 1)
    with pytest.raises(RuntimeError, match="the cache is on device"):
        write()
