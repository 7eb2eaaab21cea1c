"""Calls for many tokens of several sequences against plain statements in 64 bits: head norms with rotation, the paged cache with its attention and
copies, the delta rule, and a layer of them together.

u = 2^-24 is half a step of fp32.  Each tolerance counts the roundings between the inputs and an output.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def ints(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def starts(new):
    return [0, *np.cumsum(new).tolist()]


@pytest.fixture(autouse=True)
def status_is_clear(gpu):
    yield
    try:
        assert gpu.device_status() == 0
    finally:
        gpu.clear_status()


# ---- head norms and rotation ------------------------------------------------------------------------------
def turned(x, w, pos, freq, n_rot, eps):
    """In 64 bits, and what an output's error is measured by: the largest of the two values that were turned into each other."""
    import torch
    x = x.double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    size = x.abs().clone()
    if n_rot:
        h = n_rot // 2
        a = (pos.double()[:, None] * freq)[:, None]
        c, s = a.cos(), a.sin()
        p, q = x[..., :h].clone(), x[..., h:n_rot].clone()
        x[..., :h], x[..., h:n_rot] = p * c - q * s, q * c + p * s
        size[..., :h] = size[..., h:n_rot] = p.abs() + q.abs()
    return x, size


# roundings of an output: the sum of squares 11 deep, halved by the root, with mean, eps, root and division 4 more: 10; two products: 12.  Turned: the angle is
# rounded once (at most pi u), the sine is within 2 steps (4 u), a product and a fused add: 12 + 3.2 + 4 + 2 of |a| + |b|
QK_ROUNDINGS = 22


@pytest.mark.parametrize("n_tok,n_head,n_head_kv,dim,n_rot", [
    (1, 24, 4, 256, 64), (1, 1, 1, 256, 256), (7, 24, 4, 256, 64), (200, 24, 4, 256, 64), (33, 8, 8, 128, 128), (5, 3, 1, 64, 62), (3, 40, 8, 100, 20),
    (2, 5, 2, 33, 0), (9, 2, 1, 1, 0), (4, 6, 3, 254, 2), (17, 0, 4, 256, 64), (17, 24, 0, 256, 64), (1300, 4, 2, 36, 8)])
@pytest.mark.parametrize("layout", ["packed", "beside a gate", "odd", "in place"])
def test_head_norms(gpu, n_tok, n_head, n_head_kv, dim, n_rot, layout):
    import torch
    g = torch.Generator(device="cuda").manual_seed(n_tok * 1000 + dim)
    wide, odd = {"beside a gate": (2 * dim, 0), "odd": (dim + 3, 1)}.get(layout, (dim, 0))

    def rows(heads):
        x = torch.randn(n_tok * heads * wide + odd, generator=g, device="cuda")[odd:].reshape(n_tok, heads, wide)
        return x * torch.exp(4 * torch.randn(n_tok, heads, 1, generator=g, device="cuda"))
    q, k = rows(n_head), rows(n_head_kv)
    wq, wk = (1 + 0.3 * torch.randn(dim + odd, generator=g, device="cuda")[odd:] for _ in range(2))
    pos = torch.randint(0, 262144, (n_tok,), generator=g, device="cuda", dtype=torch.int32)
    pos[0] = 262143
    if n_tok > 3:
        pos[1], pos[2], pos[3] = 0, -5, 2 ** 31 - 1
    freq = 1e7 ** (-torch.arange(n_rot // 2, dtype=torch.float64, device="cuda") / max(1, n_rot // 2))
    q_want, k_want = turned(q[..., :dim], wq, pos, freq, n_rot, 1e-6), turned(k[..., :dim], wk, pos, freq, n_rot, 1e-6)
    empty = lambda h: torch.full((n_tok * h * dim + odd,), 7.0, device="cuda")[odd:].reshape(n_tok, h, dim)  # noqa: E731
    q_out, k_out = (q, k) if layout == "in place" else (empty(n_head), empty(n_head_kv))
    args = (n_tok, n_head, n_head_kv, dim, n_rot, n_head * wide, wide, n_head_kv * wide, wide, 1e-6)
    assert gpu.qk_norm_rope(q, k, wq, wk, pos, freq, q_out, k_out, *args) == 0
    for got, (want, size) in ((q_out, q_want), (k_out, k_want)):
        assert bool(((got.double() - want).abs() <= QK_ROUNDINGS * U * size).all())


def test_head_norms_of_a_view(gpu):
    """Strides come from the call: heads first, then tokens."""
    import torch
    n, h, d = 6, 4, 64
    x = torch.randn(h, n, d, device="cuda")
    w, out = torch.ones(d, device="cuda"), torch.empty(n, h, d, device="cuda")
    none = torch.empty(0, device="cuda")
    v = x.transpose(0, 1)
    assert gpu.qk_norm_rope(v, none, w, w, None, None, out, none, n, h, 0, d, 0, d, n * d, 0, 0, 1e-6) == 0
    want, size = turned(v, w, None, None, 0, 1e-6)
    assert bool(((out.double() - want).abs() <= QK_ROUNDINGS * U * size).all())


def test_head_norms_of_odd_values(gpu):
    """A row of zeros stays zeros; an infinity or NaN stays in its row."""
    import torch
    x = torch.randn(3, 2, 64, device="cuda")
    x[0, 0], x[1, 1, 3], x[2, 0, 5] = 0.0, math.inf, math.nan
    w, out, none = torch.ones(64, device="cuda"), torch.empty(3, 2, 64, device="cuda"), torch.empty(0, device="cuda")
    freq = torch.ones(16, dtype=torch.float64, device="cuda")
    assert gpu.qk_norm_rope(x, none, w, w, ints([1, 2, 3]), freq, out, none, 3, 2, 0, 64, 32, 128, 64, 0, 0, 1e-6) == 0
    assert bool((out[0, 0] == 0).all()) and bool(out[1, 1].isnan().any()) and bool(out[2, 0].isnan().all())
    assert bool(out[0, 1].isfinite().all() and out[1, 0].isfinite().all() and out[2, 1].isfinite().all())


# ---- the paged cache ---------------------------------------------------------------------------------------
def q8_0(x):
    """Codes and scales (numpy): scale = largest magnitude times 1 / 127 in fp32, codes by its reciprocal, halves away from zero; the scale as fp16, halves away."""
    x = np.ascontiguousarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        d = np.max(np.abs(x), -1) * (np.float32(1) / np.float32(127))
        inv = np.where(d > 0, np.float32(1) / d, np.float32(0)).astype(np.float32)
        t = (x * inv[..., None]).astype(np.float32).astype(np.float64)
        t = np.where(np.isnan(t), 0.0, t)
        codes = np.clip(np.sign(t) * np.floor(np.abs(t) + 0.5), -127, 127).astype(np.int8)
        e = np.maximum(np.frexp(d.astype(np.float64))[1] - 1, -14)
        step = np.ldexp(1.0, e - 10)
        half = np.where(np.isinf(d), np.inf, np.floor(d / step + 0.5) * step)
        return codes, half.astype(np.float16)


def blocks(x):
    codes, d = q8_0(x)
    return np.concatenate([d[..., None].view(np.uint8), codes.view(np.uint8)], -1)


def number(b):
    b = np.ascontiguousarray(b)
    with np.errstate(all="ignore"):
        return (b[..., 2:].view(np.int8).astype(np.float64) * b[..., :2].copy().view(np.float16).astype(np.float64)).reshape(*b.shape[:-2], -1)


class Cache:
    """A pool of random rows, pages in random order, and the library's view of it."""

    def __init__(self, gpu, lens, new, n_layers=1, n_head_kv=4, seed=0, spare=2, behind=0, scale=1.0):
        import torch
        rng = np.random.default_rng(seed)
        used = [-(-n // 64) for n in lens]
        self.n_pages, self.lens, self.new, self.hkv = sum(used) + spare, lens, new, n_head_kv
        order = rng.permutation(self.n_pages)
        stride = max(1, max(used)) + 1
        self.table = np.full((len(lens), stride), -1, np.int32)            # what is behind a sequence's pages is never looked at
        at = 0
        for i, u in enumerate(used):
            self.table[i, :u] = order[at:at + u]
            at += u
        x = rng.standard_normal((self.n_pages, n_layers, 2, n_head_kv, 64, 256)).astype(np.float32) * np.float32(scale)
        self.pool = blocks(x)
        self.n_tok = sum(new) + behind
        self.start = starts(new)
        self.d_pool = torch.from_numpy(self.pool).cuda()
        self.view = gpu.Pages(self.d_pool, ints(self.table), ints(lens), ints(self.start), n_layers, n_head_kv, self.n_tok)

    def upload(self):
        import torch
        self.d_pool.copy_(torch.from_numpy(self.pool))

    def rows(self, s, layer, kv, head):
        """The rows of a sequence as numbers, [positions][256]."""
        n = self.lens[s]
        if n == 0:
            return np.zeros((0, 256))
        return number(self.pool[self.table[s, :-(-n // 64)], layer, kv, head].reshape(-1, 8, 34)[:n])


def run_attention(gpu, c, q, layer=0, max_len=None, scale=0.0625):
    import torch
    n_head, max_len = q.shape[1], max_len or max(1, max(c.lens))
    out = torch.full_like(q, 7.0)
    size = c.view.attn_workspace(max_len, n_head)
    ws = torch.full((size // 4,), math.nan, device="cuda") if size else None
    assert c.view.attn(layer, q, out, n_head, max_len, ws, scale) == 0
    return out


def attention(c, q, layer=0, scale=0.0625):
    """Each token by itself in 64 bits; rows of nobody 7.  With it the size of an output's error: sum of p |v|, and the largest sum of |q k| (scaled)."""
    q = q.cpu().numpy()
    n_head, group = q.shape[1], q.shape[1] // c.hkv
    out, size = np.full(q.shape, 7.0), np.zeros(q.shape)
    codes, d = q8_0(q)
    qn = (codes.astype(np.float64) * d[..., None].astype(np.float64)).reshape(q.shape)
    for s, n in enumerate(c.new):
        for h in range(n_head if n else 0):
            k, v = c.rows(s, layer, 0, h // group), c.rows(s, layer, 1, h // group)
            for t in range(n):
                row, see = c.start[s] + t, c.lens[s] - n + t + 1
                if see <= 0:
                    out[row, h] = 0.0
                    continue
                with np.errstate(all="ignore"):
                    x = k[:see] @ qn[row, h] * scale
                    p = np.exp(x - np.max(x))
                    p /= p.sum()
                    out[row, h] = p @ v[:see]
                    big = np.max(np.abs(k[:see]) @ np.abs(qn[row, h])) * abs(scale)
                    size[row, h] = (1 + big) * (p @ np.abs(v[:see]))
    return out, size


# Roundings.  A score is a sum of 8 terms of two rounded products each, beside the query's scale times the softmax's: 11 u of the sum of |q k|, and what it is
# off by every weight is off by.  A weight: subtraction (u of the scores' distance, at most 2 of the sum), expf 2 steps (4 u), scale 1, planes 2^-22 (4 u); sums of 16
# products cut off to 2^-23 a step, 8 steps a page (16 u); per page two roundings of the output, pages in a tree of splits.  Weights' sum 10, division and products 5.
def attn_bound(size, n_pages):
    return size * U * (48 + 2 * n_pages)


def close(got, want, size, n_pages):
    err = np.abs(got.double().cpu().numpy() - want)
    over = err - attn_bound(size, n_pages)
    assert not np.isnan(over).any() and over.max() <= 0, f"off by {err.max():.3e}, {np.max(err / np.maximum(attn_bound(size, n_pages), 1e-300)):.2f} of the bound"


@pytest.mark.parametrize("lens,new,n_head_kv,behind", [
    ([1], [1], 4, 0), ([64], [64], 4, 0), ([65], [2], 1, 3), ([200, 3, 64, 0, 129], [70, 3, 1, 0, 0], 4, 2), ([700] * 40, [5] * 40, 2, 0), ([130], [128], 3, 0)])
@pytest.mark.parametrize("offset", [0, 1])
def test_append(gpu, lens, new, n_head_kv, behind, offset):
    """The bytes of the new rows; every other byte as it was."""
    import torch
    c = Cache(gpu, lens, new, n_layers=2, n_head_kv=n_head_kv, behind=behind, seed=len(lens))
    rng = np.random.default_rng(3)
    k, v = (rng.standard_normal((c.n_tok, n_head_kv, 256)).astype(np.float32) * np.exp(3 * rng.standard_normal((c.n_tok, 1, 1))).astype(np.float32) for _ in range(2))
    k[0, 0, :32], v[0, 0, 32:64], k[0, 0, 70] = 0.0, 1e-7, 1e6             # zeros; a subnormal scale; one past fp16's largest
    flat = lambda x: torch.cat([torch.zeros(offset), torch.from_numpy(x).flatten()]).cuda()[offset:]  # noqa: E731
    assert c.view.append(1, flat(k), flat(v)) == 0
    want = c.pool.copy()
    for s, n in enumerate(new):
        for t in range(n):
            p, row = lens[s] - n + t, c.start[s] + t
            want[c.table[s, p // 64], 1, 0, :, p % 64], want[c.table[s, p // 64], 1, 1, :, p % 64] = blocks(k[row]), blocks(v[row])
    assert np.array_equal(c.d_pool.cpu().numpy(), want)


CASES = [  # lengths, new tokens, query heads, kv heads, rows of nobody
    ([1], [1], 24, 4, 0), ([64], [1], 24, 4, 0), ([65], [1], 24, 4, 0), ([2000], [1], 24, 4, 0), ([700], [5], 24, 4, 0), ([130], [130], 24, 4, 1), ([64], [64], 8, 8, 0),
    ([300], [21], 6, 6, 0), ([300], [40], 8, 1, 0), ([129], [7], 5, 1, 0), ([90, 1, 0, 640, 64, 63], [9, 1, 0, 70, 0, 63], 24, 4, 4), ([33] * 50, [1] * 50, 4, 2, 0),
    ([900, 40], [200, 40], 12, 2, 0), ([17] * 3, [3] * 3, 16, 1, 0), ([2000], [100], 24, 4, 0), ([700, 9], [600, 2], 2, 2, 0), ([1200, 64, 3000], [90, 8, 1], 24, 4, 5),
    ([300], [24], 32, 1, 0), ([130, 140], [3, 2], 9, 3, 0), ([3000], [2], 16, 8, 0)]


@pytest.mark.parametrize("lens,new,n_head,n_head_kv,behind", CASES)
def test_attention(gpu, lens, new, n_head, n_head_kv, behind):
    import torch
    c = Cache(gpu, lens, new, n_layers=2, n_head_kv=n_head_kv, behind=behind, seed=sum(lens))
    q = torch.randn(c.n_tok, n_head, 256, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    want, size = attention(c, q, layer=1)
    close(run_attention(gpu, c, q, layer=1), want, size, -(-max(lens) // 64))


@pytest.mark.parametrize("max_len", [1, 100, 5000, 262144])
def test_attention_by_any_division(gpu, max_len):
    """max_len divides the work, and no more: too small a one as well."""
    import torch
    c = Cache(gpu, [1500, 70], [3, 70], seed=1)
    q = torch.randn(c.n_tok, 24, 256, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")
    want, size = attention(c, q)
    close(run_attention(gpu, c, q, max_len=max_len), want, size, 24)


@pytest.mark.parametrize("new", [[1, 1], [90, 3]])
def test_attention_of_odd_offsets(gpu, new):
    import torch
    c = Cache(gpu, [200, 100], new, seed=2)
    base = torch.randn(c.n_tok * 24 * 256 + 1, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
    q = base[1:].reshape(c.n_tok, 24, 256)
    out = torch.zeros(c.n_tok * 24 * 256 + 1, device="cuda")[1:].reshape(c.n_tok, 24, 256)
    size = c.view.attn_workspace(200, 24)
    assert c.view.attn(0, q, out, 24, 200, torch.empty(size, dtype=torch.uint8, device="cuda") if size else None, 0.0625) == 0
    assert torch.equal(out, run_attention(gpu, c, q.clone()))


@pytest.mark.parametrize("new", [1, 3, 100])
def test_attention_of_values_far_apart(gpu, new):
    """Scales of values that lie 2^22 apart within a page: the small ones keep their digits where the large ones have no weight."""
    import torch
    c = Cache(gpu, [200], [new], seed=4)
    pool = c.pool.copy()
    scale = pool[..., :2].copy().view(np.float16)[..., 0]
    scale[:, 0, 1] = np.where(np.arange(64)[:, None] % 7 == 0, np.float16(60.0), np.float16(2e-5))           # V of every seventh row
    scale[:, 0, 0] = np.float16(0.01)
    pool[..., :2] = scale[..., None].view(np.uint8)
    pool[:, 0, 0, :, ::7, :, 2:] = np.int8(-127).view(np.uint8)                # ... whose K points away from the query
    pool[:, 0, 0, :, 1::7, :, 2:] = np.int8(100).view(np.uint8)
    c.pool = pool
    c.upload()
    q = torch.ones(c.n_tok, 24, 256, device="cuda")
    want, size = attention(c, q)
    assert np.abs(want).max() < 0.1                    # 2^-5 of a large value, 2^22 times what the large ones are weighted by
    close(run_attention(gpu, c, q), want, size, 4)


def test_nothing_hidden_reaches_a_row(gpu):
    """Infinities and NaN in rows behind the last position and in those of later tokens; a token that sees one has it."""
    import torch
    for new in (3, 150):
        c = Cache(gpu, [230], [new], seed=8)
        q = torch.randn(c.n_tok, 24, 256, generator=torch.Generator(device="cuda").manual_seed(8), device="cuda")
        want, size = attention(c, q)
        for what in (np.float16(np.inf), np.float16(np.nan)):
            pool = c.pool.copy()
            bad = np.frombuffer(what.tobytes(), np.uint8)
            last = 229                                  # the last token's own row, in V and in K of another head
            pool[c.table[0, last // 64], 0, 1, 0, last % 64, :, :2] = bad
            pool[c.table[0, last // 64], 0, 0, 1, last % 64, :, :2] = bad
            for p in range(230, 256):
                pool[c.table[0, p // 64], 0, :, :, p % 64, :, :2] = bad
            c.d_pool.copy_(torch.from_numpy(pool))
            out = run_attention(gpu, c, q)
            # (a page that holds such a value is multiplied in another way, for the rows that do not see it too: other bits, the same bound)
            close(out[:-1], want[:-1], size[:-1], 4)
            close(out[-1, 12:], want[-1, 12:], size[-1, 12:], 4)
            assert bool((~out[-1, :12].isfinite()).all())


@pytest.mark.parametrize("lens,new", [([3, 0, 70], [5, 4, 70]), ([10, 0], [150, 30]), ([1], [2])])
def test_tokens_without_a_position_see_nothing(gpu, lens, new):
    import torch
    c = Cache(gpu, lens, new, seed=9)
    q = torch.randn(c.n_tok, 24, 256, device="cuda")
    want, size = attention(c, q)
    out = run_attention(gpu, c, q)
    close(out, want, size, 2)
    for s, n in enumerate(new):
        none = slice(c.start[s], c.start[s] + max(0, n - lens[s]))
        assert (want[none] == 0).all() and bool((out[none] == 0).all())


def test_rows_that_several_sequences_claim(gpu):
    """Starts that run over each other's rows: whatever becomes of those rows, nothing else is touched."""
    import torch
    c = Cache(gpu, [400, 400, 400], [150, 150, 100], seed=14)
    start = c.view._keep[3]
    start.copy_(ints([0, 400, 0, 400]))
    q = torch.randn(c.n_tok, 24, 256, device="cuda")
    before = c.d_pool.clone()
    run_attention(gpu, c, q)
    torch.cuda.synchronize()
    assert torch.equal(before, c.d_pool)
    args = delta_inputs(200, 2, 6, 128, 128, 3)
    state = torch.zeros(3, 6, 128, 128, device="cuda")
    size = gpu.gdn_seqs_workspace(200, 3, 2, 6, 128, 128)
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
    out = torch.zeros(200, 6, 128, device="cuda")
    assert gpu.gdn_seqs(state, *args, out, ints([0, 200, 0, 200]), None, ws, size, 3, 3, 200, 2, 6, 128, 128) == 0
    gpu.device_status()
    gpu.clear_status()


@pytest.mark.parametrize("new,max_len", [([2, 2, 2], 300), ([2, 2, 2], 20000), ([100, 2, 2], 300)])
def test_numbers_that_do_not_fit_stop_their_sequence(gpu, new, max_len):
    """A page that the pool does not have, a length past the table, rows outside the call: the others are served, the status word says so."""
    import torch
    c = Cache(gpu, [300, 200, 150], new, seed=10)
    q = torch.randn(c.n_tok, 24, 256, device="cuda")
    k, v = torch.randn(c.n_tok, 4, 256, device="cuda"), torch.randn(c.n_tok, 4, 256, device="cuda")
    assert c.view.append(0, k, v) == 0
    after = c.d_pool.clone()
    clean = run_attention(gpu, c, q, max_len=max_len)
    table, length, start = c.view._keep[1:]
    a, b = new[0], new[0] + new[1]

    def check(keep_first_middle):
        c.d_pool.copy_(torch.from_numpy(c.pool))
        assert gpu.clear_status() == 0 and c.view.append(0, k, v) == 0
        assert gpu.device_status() == 3 and gpu.clear_status() == 0
        mine = after.clone()
        mine[ints(c.table[1, :4]).long()] = torch.from_numpy(c.pool).cuda()[ints(c.table[1, :4]).long()]
        assert torch.equal(c.d_pool, mine)
        c.d_pool.copy_(after)
        out = run_attention(gpu, c, q, max_len=max_len)
        assert gpu.device_status() == 3 and gpu.clear_status() == 0
        assert torch.equal(out[:a], clean[:a]) and torch.equal(out[b:], clean[b:])
        if keep_first_middle:
            assert bool((out[a:b] == 7).all())
    for page in (-1, c.n_pages, 2 ** 31 - 1, -2 ** 31):
        table[1, 3] = page                              # the page of the new tokens
        check(False)
    table.copy_(ints(c.table))
    for n in (6 * 64 + 1, 2 ** 31 - 1):
        length[1] = n
        check(True)
    length[1] = 200
    start[2], start[3] = a - 1, 2 ** 31 - 1             # rows that run backwards, and past the call
    out = run_attention(gpu, c, q, max_len=max_len)
    assert torch.equal(out[:a], clean[:a]) and bool((out[a:] == 7).all())
    assert gpu.device_status() == 3 and gpu.clear_status() == 0


def test_rows_that_run_backwards_are_reported(gpu):
    """Starts of which one sequence's run backwards, and no row is left to it: the status word says so, in every call."""
    import torch
    c = Cache(gpu, [300, 200, 150], [3, 3, 3], seed=15)
    c.view._keep[3].copy_(ints([0, 5, 3, 9]))
    q = torch.randn(c.n_tok, 24, 256, device="cuda")
    k, v = torch.randn(c.n_tok, 4, 256, device="cuda"), torch.randn(c.n_tok, 4, 256, device="cuda")
    assert gpu.clear_status() == 0 and c.view.append(0, k, v) == 0
    assert gpu.device_status() == 3 and gpu.clear_status() == 0
    run_attention(gpu, c, q)
    assert gpu.device_status() == 3 and gpu.clear_status() == 0
    args = delta_inputs(9, 2, 6, 128, 128, 3)
    state, out = torch.zeros(3, 6, 128, 128, device="cuda"), torch.zeros(9, 6, 128, device="cuda")
    assert gpu.gdn_seqs(state, *args, out, ints([0, 5, 3, 9]), None, None, 0, 3, 3, 9, 2, 6, 128, 128) == 0
    assert gpu.device_status() == 3 and gpu.clear_status() == 0


def test_rows_that_many_sequences_claim(gpu):
    """64 sequences of which every other one claims all rows: no more work than the call's rows can be, and nothing outside the outputs is written."""
    import torch
    c = Cache(gpu, [70] * 64, [2] * 64, seed=16)
    c.view._keep[3].copy_(ints([0, 128] * 32 + [0]))
    q = torch.randn(c.n_tok, 24, 256, device="cuda")
    before = c.d_pool.clone()
    out = run_attention(gpu, c, q)
    torch.cuda.synchronize()
    assert torch.equal(before, c.d_pool) and bool(torch.isfinite(out).all())
    assert gpu.device_status() == 3 and gpu.clear_status() == 0


def test_cache_of_another_device(gpu, monkeypatch):
    """The numbers of a cache are memory of its own device: a call on another one is refused."""
    import torch
    c = Cache(gpu, [70, 20], [2, 2], seed=17)
    q = torch.randn(c.n_tok, 24, 256, device="cuda")
    k = torch.randn(c.n_tok, 4, 256, device="cuda")
    monkeypatch.setattr(c.view, "_device", c.view._device + 1)
    with pytest.raises(RuntimeError, match="the cache is on device"):
        c.view.append(0, k, k)
    with pytest.raises(RuntimeError, match="the cache is on device"):
        c.view.attn(0, q, torch.empty_like(q), 24, 70, None, 0.0625)


def test_captured_attention_follows_the_numbers(gpu):
    """A captured step is replayed with other lengths, rows and pages."""
    import torch
    c = Cache(gpu, [700, 300], [2, 3], seed=11, spare=20)
    q, k, v = torch.randn(5, 24, 256, device="cuda"), torch.randn(5, 4, 256, device="cuda"), torch.randn(5, 4, 256, device="cuda")
    out = torch.empty_like(q)
    ws = torch.empty(c.view.attn_workspace(1000, 24), dtype=torch.uint8, device="cuda")
    step = lambda: c.view.append(0, k, v) or c.view.attn(0, q, out, 24, 1000, ws, 0.0625)  # noqa: E731
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(st):
        assert step() == 0
        with torch.cuda.graph(graph, stream=st):
            assert step() == 0
    torch.cuda.synchronize()
    table, length, start = c.view._keep[1:]
    for lens, new in (([704, 301], [4, 1]), ([640, 64], [0, 5]), ([65, 1], [1, 1])):
        c.d_pool.copy_(torch.from_numpy(c.pool))
        length.copy_(ints(lens))
        start.copy_(ints(starts(new)))
        q.normal_()
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        got, pool = out.clone(), c.d_pool.clone()
        c.d_pool.copy_(torch.from_numpy(c.pool))
        out.fill_(7.0)
        assert step() == 0
        assert torch.equal(got, out) and torch.equal(pool, c.d_pool)
        assert bool((out[sum(new):] == 7).all())


def test_attention_repeats_its_bits_on_other_streams(gpu):
    import torch
    c = Cache(gpu, [3000, 100], [2, 90], seed=12)
    q = torch.randn(c.n_tok, 24, 256, device="cuda")
    first = run_attention(gpu, c, q)
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        with torch.cuda.stream(torch.cuda.Stream()):
            outs.append(run_attention(gpu, c, q))
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)


@pytest.mark.parametrize("n_pages,page_bytes,moved", [(5, 16, 2), (9, 32 * 1024 + 16, 4), (1100, 4352, 500), (40, 139264, 17)])
def test_copies(gpu, n_pages, page_bytes, moved):
    import torch
    rng = np.random.default_rng(n_pages)
    pool = torch.from_numpy(rng.integers(0, 256, (n_pages, page_bytes), dtype=np.uint8)).cuda()
    order = torch.from_numpy(rng.permutation(n_pages).astype(np.int32))
    src, dst = order[:moved].clone(), order[moved:2 * moved].clone()
    src[1] = src[0]                                     # one page to two places
    want = pool.clone()
    want[dst.long().cuda()] = pool[src.long().cuda()]
    assert gpu.pages_copy(pool, page_bytes, n_pages, src, dst, moved) == 0
    assert torch.equal(pool, want)
    with pytest.raises(RuntimeError, match="shorter"):
        gpu.pages_copy(pool, page_bytes, n_pages, src, dst, moved + 1)
    with pytest.raises(RuntimeError, match="host memory"):
        gpu.pages_copy(pool, page_bytes, n_pages, src.cuda(), dst, moved)
    assert gpu.pages_copy(pool, page_bytes, n_pages, src, src, moved) == 1 and torch.equal(pool, want)


def test_views_that_are_refused(gpu):
    import torch
    pool, table, length, start = torch.zeros(2, 2 * 17408, dtype=torch.uint8, device="cuda"), ints([[0]]), ints([1]), ints([0, 1])
    gpu.Pages(pool, table, length, start, 1, 1, 1)
    for args in ((pool.float(), table, length, start, 1, 1, 1), (pool, table.long(), length, start, 1, 1, 1), (pool, table, length, start, 1, 3, 1),
                 (pool, table, length, start, 0, 1, 1), (pool, table, ints([1, 1]), start, 1, 1, 1), (pool, table, length, ints([0, 1, 2]), 1, 1, 1),
                 (pool, table[0], length, start, 1, 1, 1), (pool.t(), table, length, start, 1, 1, 1), (pool.cpu(), table, length, start, 1, 1, 1)):
        with pytest.raises(RuntimeError):
            gpu.Pages(*args)


# ---- the delta rule --------------------------------------------------------------------------------------
def delta_inputs(n_tok, kh, vh, K, V, seed, decay=0.3):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
    return (unit(normal(n_tok, kh, K)) * K ** -0.5, unit(normal(n_tok, kh, K)), normal(n_tok, vh, V), -decay * normal(n_tok, vh).abs(),
            torch.sigmoid(normal(n_tok, vh)))


def delta(state, q, k, v, g, beta, start, slots):
    """Token by token in 64 bits: outputs (rows of nobody 7), states."""
    import torch
    out, state = torch.full(v.shape, 7.0, dtype=torch.float64, device="cuda"), state.double()
    share = v.shape[1] // k.shape[1]
    for s in range(len(start) - 1):
        S = state[slots[s]]
        for t in range(start[s], start[s + 1]):
            S = S * g[t].double().exp()[:, None, None]
            kt, qt = k[t].double().repeat_interleave(share, 0), q[t].double().repeat_interleave(share, 0)
            miss = v[t].double() - torch.einsum("hk,hkv->hv", kt, S)
            S = S + torch.einsum("hk,hv,h->hkv", kt, miss, beta[t].double())
            out[t] = torch.einsum("hk,hkv->hv", qt, S)
        state[slots[s]] = S
    return out, state


def run_delta(gpu, state, args, new, slots=None, behind=0):
    import torch
    q, k, v, g, beta = args
    out = torch.full_like(v, 7.0)
    n_tok, kh, K = k.shape
    vh, V = v.shape[1:]
    size = gpu.gdn_seqs_workspace(n_tok, len(new), kh, vh, K, V)
    ws = torch.full((size // 4,), math.nan, device="cuda") if size else None
    rc = gpu.gdn_seqs(state, q, k, v, g, beta, out, ints(starts(new)), None if slots is None else ints(slots), ws, size, len(new), state.shape[0], n_tok, kh, vh, K, V)
    assert rc == 0
    return out


# The bound of bonsai_p40_gdn_step, and of one recurrent step after the other (3e-5 of the largest after three there): unit keys and steps below one keep an error from
# growing, each token adds one of about 10 roundings of sums of K products, u sqrt(10 K): 2e-6; 40 of them side by side, of a state that forgets.
DELTA_TOL = 1e-5


def near(got, want):
    err, size = (got.double() - want).abs().max().item(), want.abs().max().item()
    assert err <= DELTA_TOL * size, f"off by {err:.3e} of {size:.3e}"


DELTA = [  # new tokens, key heads, value heads, K, V
    ([1], 16, 48, 128, 128), ([5], 16, 48, 128, 128), ([1, 0, 3, 2], 16, 48, 128, 128), ([63], 2, 6, 128, 128), ([64], 2, 6, 128, 128), ([65], 2, 2, 128, 128), ([200], 1, 3, 128, 128),
    ([130, 1, 0, 64, 17, 300], 2, 6, 128, 128), ([700], 16, 48, 128, 128), ([3, 90], 2, 4, 64, 32), ([40], 1, 2, 128, 96), ([70], 2, 2, 100, 64), ([9], 1, 1, 1, 32), ([33, 31, 16, 15], 4, 4, 128, 128)]


@pytest.mark.parametrize("new,kh,vh,K,V", DELTA)
def test_delta(gpu, new, kh, vh, K, V):
    import torch
    behind = 3
    args = delta_inputs(sum(new) + behind, kh, vh, K, V, sum(new))
    state = torch.randn(len(new), vh, K, V, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") * 0.1
    want, S = delta(state, *args, starts(new), range(len(new)))
    out = run_delta(gpu, state, args, new)
    near(out[:sum(new)], want[:sum(new)])
    near(state, S)
    assert bool((out[sum(new):] == 7).all())


@pytest.mark.parametrize("new", [[3, 2, 1], [70, 2, 130]])
def test_delta_slots(gpu, new):
    """States by slots; those of nobody stay as they are, and so do the states of two sequences that name the same one, or none of the pool."""
    import torch
    args = delta_inputs(sum(new), 2, 6, 128, 128, 3)
    state = torch.randn(7, 6, 128, 128, device="cuda") * 0.1
    want, S = delta(state, *args, starts(new), [5, 0, 3])
    was = state.clone()
    out = run_delta(gpu, state, args, new, [5, 0, 3])
    near(out, want)
    near(state, S)
    for s in (1, 2, 4, 6):
        assert torch.equal(state[s], was[s])
    for slots, served in (([5, 5, 3], 3), ([7, -1, 3], 3)):
        state.copy_(was)
        out = run_delta(gpu, state, args, new, slots)
        assert gpu.device_status() == 3 and gpu.clear_status() == 0
        near(state[served], S[served])
        assert bool((out[:new[0] + new[1]] == 7).all())
        state[served] = was[served]
        assert torch.equal(state, was)


@pytest.mark.parametrize("new", [[6], [150]])
@pytest.mark.parametrize("case", ["forgets at once", "forgets nothing", "resets", "same keys", "no steps", "grows", "large"])
def test_delta_extremes(gpu, new, case):
    import torch
    q, k, v, g, beta = delta_inputs(new[0], 1, 3, 128, 128, 17)
    state = torch.randn(1, 3, 128, 128, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    if case == "forgets at once":
        g -= 30.0
    elif case == "forgets nothing":
        g.zero_()
    elif case == "resets":
        g[new[0] // 2] = -math.inf
        g[new[0] - 1, 1] = -1e30
    elif case == "same keys":
        k[:] = k[0]
        beta.fill_(1.0)
    elif case == "no steps":
        beta.zero_()
    elif case == "grows":
        g.neg_().mul_(0.5)
    else:
        v *= 1e20
        state *= 1e20
    want, S = delta(state, q, k, v, g, beta, [0, new[0]], [0])
    out = run_delta(gpu, state, (q, k, v, g, beta), new)
    near(out, want)
    near(state, S)


def test_delta_in_pieces(gpu):
    """A prompt at once and in pieces, single tokens among them."""
    import torch
    args = delta_inputs(300, 16, 48, 128, 128, 23)
    a = torch.randn(1, 48, 128, 128, device="cuda") * 0.1
    b = a.clone()
    whole, at, parts = run_delta(gpu, a, args, [300]), 0, []
    for n in (1, 100, 64, 3, 132):
        parts.append(run_delta(gpu, b, [x[at:at + n] for x in args], [n]))
        at += n
    near(torch.cat(parts), whole.double())
    near(b, a.double())
    step = torch.empty(48, 128, device="cuda")
    c = a.clone()
    q, k, v, g, beta = (x[:1].contiguous() for x in args)
    one = run_delta(gpu, a, (q, k, v, g, beta), [1])
    assert gpu.gdn_step(c, q, k, v, g, beta, step, 16, 48, 128, 128) == 0
    near(one[0], step.double())
    near(a[0], c[0].double())


def test_delta_repeats_its_bits(gpu):
    import torch
    args = delta_inputs(200, 16, 48, 128, 128, 29)
    first = None
    for _ in range(3):
        state = torch.full((2, 48, 128, 128), 0.01, device="cuda")
        out = run_delta(gpu, state, args, [130, 70])
        if first is None:
            first = out, state
        assert torch.equal(out, first[0]) and torch.equal(state, first[1])


# ---- a run of them together -----------------------------------------------------------------------------------
def test_a_layer_in_chunks_forks_and_compacted(gpu):
    """Norm, rotation, append and attention of a prompt in chunks, token by token behind a fork, after a compaction: the same outputs as all tokens at once."""
    import torch
    from bonsai_b200.pages import PageBook
    H, HKV, D, N, PAGES = 24, 4, 256, 150, 12
    gen = torch.Generator(device="cuda").manual_seed(31)
    proj = torch.randn(N, H, 2 * D, generator=gen, device="cuda")
    kx, vx = torch.randn(N, HKV, D, generator=gen, device="cuda"), torch.randn(N, HKV, D, generator=gen, device="cuda")
    wq, wk = torch.ones(D, device="cuda"), torch.ones(D, device="cuda")
    freq = 1e7 ** (-torch.arange(32, dtype=torch.float64, device="cuda") / 32)
    pool = torch.zeros(PAGES, 2 * HKV * 64 * 272, dtype=torch.uint8, device="cuda")
    book = PageBook(PAGES)

    def copies(src, dst):
        if src:
            assert gpu.pages_copy(pool, pool.shape[1], PAGES, torch.tensor(src, dtype=torch.int32), torch.tensor(dst, dtype=torch.int32), len(src)) == 0

    def step(rows):
        """rows: {sequence: its tokens of the text}."""
        for s, r in rows.items():
            copies(*book.extend(s, len(r)))
        at = torch.cat([torch.tensor(list(r)) for r in rows.values()]).cuda()
        n = len(at)
        q, k = torch.empty(n, H, D, device="cuda"), torch.empty(n, HKV, D, device="cuda")
        p, kk, vv = proj[at].contiguous(), kx[at].contiguous(), vx[at].contiguous()
        assert gpu.qk_norm_rope(p, kk, wq, wk, at.int(), freq, q, k, n, H, HKV, D, 64, H * 2 * D, 2 * D, HKV * D, D, 1e-6) == 0
        table, lens = book.tables(list(rows))
        view = gpu.Pages(pool, ints(table), ints(lens), ints(starts([len(r) for r in rows.values()])), 1, HKV, n)
        assert view.append(0, k, vv) == 0
        out, size = torch.empty_like(q), view.attn_workspace(max(lens), H)
        assert view.attn(0, q, out, H, max(lens), torch.empty(size, dtype=torch.uint8, device="cuda") if size else None, D ** -0.5) == 0
        return out

    whole = book.new()
    want = step({whole: range(N)})
    assert bool(want.isfinite().all())
    book.free(whole)
    same = lambda got, rows: (got - want[rows]).abs().max().item() <= 1e-5 * want.abs().max().item()  # noqa: E731
    filler = book.new()
    copies(*book.extend(filler, 130))
    a = book.new()
    assert same(step({a: range(70)}), slice(0, 70))
    b = book.fork(a)
    out = step({b: range(70, 75), a: range(70, 71)})             # both write to what was one page
    assert same(out[:5], slice(70, 75)) and same(out[5:], slice(70, 71))
    book.free(filler)
    copies(*book.compact())
    assert max(book.pages(a) + book.pages(b)) == PAGES - book.free_pages - 1
    for t in range(75, 80):
        out = step({a: range(t - 4, t - 3), b: range(t, t + 1)})
        assert same(out[:1], slice(t - 4, t - 3)) and same(out[1:], slice(t, t + 1))
    book.truncate(a, 66)
    assert same(step({a: range(66, N)}), slice(66, N))
