"""How a call's attention is divided: long contexts beside prompts, many sequences, and workspaces that hold exactly what is asked for."""
import math

import numpy as np
import pytest

from test_gpu_sequences import Cache, attn_bound, number, q8_0, run_attention, status_is_clear  # noqa: F401

pytestmark = pytest.mark.gpu


def queries(c, n_head, seed=5):
    import torch
    return torch.randn(c.n_tok, n_head, 256, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def attention(c, q, layer=0, scale=0.0625):
    """Each token over the positions up to its own in 64 bits, a kv head's rows at once; rows of nobody 7.  With it the size of an output's error, as test_gpu_sequences has it."""
    import torch
    n_head, group = q.shape[1], q.shape[1] // c.hkv
    codes, d = q8_0(q.cpu().numpy())
    qn = torch.from_numpy((codes.astype(np.float64) * d[..., None].astype(np.float64)).reshape(q.shape)).cuda()
    out, size = torch.full(q.shape, 7.0, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for s, n in enumerate(c.new):
        if n == 0:
            continue
        rows, length = slice(c.start[s], c.start[s] + n), c.lens[s]
        seen = torch.arange(length, device="cuda")[None] <= torch.arange(length - n, length, device="cuda")[:, None]
        held = c.pool[c.table[s, :-(-length // 64)], layer]
        for j in range(c.hkv):
            k, v = (torch.from_numpy(number(held[:, i, j].reshape(-1, 8, 34)[:length])).cuda() for i in range(2))
            for h in range(j * group, (j + 1) * group):
                x = (qn[rows, h] @ k.T * scale).masked_fill(~seen, -math.inf)
                p = torch.softmax(x, -1)
                out[rows, h] = p @ v
                big = (qn[rows, h].abs() @ k.abs().T).masked_fill(~seen, 0.0).amax(-1, keepdim=True) * abs(scale)
                size[rows, h] = (1 + big) * (p @ v.abs())
    return out, size


def close(got, want, size, n_pages):
    over = (got.double() - want).abs() - attn_bound(size, n_pages)
    assert not bool(over.isnan().any()) and over.max().item() <= 0, f"{((got.double() - want).abs() / attn_bound(size, n_pages).clamp(min=1e-300)).max().item():.2f} of the bound"


def run_guarded(gpu, c, q, max_len):
    """The call with a workspace of exactly the bytes asked for, 4 KB of marks on either side of it and of the outputs."""
    import torch
    size, n = c.view.attn_workspace(max_len, q.shape[1]), q.numel()
    room = torch.full((size + 8192,), 0xA5, dtype=torch.uint8, device="cuda")
    room[4096:4096 + size].view(torch.float32).fill_(math.nan)
    outs = torch.full((n + 2048,), 7.0, device="cuda")
    out = outs[1024:1024 + n].reshape(q.shape)
    pool = c.d_pool.clone()
    assert c.view.attn(0, q, out, q.shape[1], max_len, room[4096:4096 + size] if size else None, 0.0625) == 0
    assert bool((room[:4096] == 0xA5).all()) and bool((room[4096 + size:] == 0xA5).all())
    assert bool((outs[:1024] == 7).all()) and bool((outs[1024 + n:] == 7).all()) and torch.equal(pool, c.d_pool)
    return out


CASES = [  # lengths, new tokens, query heads, kv heads, max_len
    ([20000, 300, 9000], [1, 200, 2], 24, 4, 20000),                           # two chats of long contexts beside a prompt: 8 rows a tile and 74 CTAs, 64 rows
    ([13000, 700, 5000, 64, 8000], [5, 600, 1, 0, 21], 24, 4, 13000),          # the same with drafted tokens (64 rows a tile)
    ([9000, 300], [2, 150], 8, 8, 9000), ([9000, 400], [3, 400], 5, 1, 9000),
    ([9000], [1], 24, 4, 9000), ([9000], [9], 24, 4, 9000), ([1500, 30], [1, 1], 64, 64, 1500), ([5000] * 3, [7] * 3, 24, 4, 5000),
    ([9000, 300], [2, 200], 24, 4, 300), ([9000, 9000], [2, 200], 24, 4, 129),         # longer than it was said to be
    ([12000, 4000, 3000], [30, 25, 60], 24, 4, 1 << 22),                       # no room for images: everything on mma.sync
    ([900, 200], [300, 200], 3, 1, 900)]


@pytest.mark.parametrize("lens,new,n_head,n_head_kv,max_len", CASES)
def test_long_contexts(gpu, lens, new, n_head, n_head_kv, max_len):
    c = Cache(gpu, lens, new, n_head_kv=n_head_kv, behind=2, seed=sum(lens))
    q = queries(c, n_head)
    want, size = attention(c, q)
    close(run_guarded(gpu, c, q, max_len), want, size, -(-max(lens) // 64))


@pytest.mark.parametrize("n_seq,each,prompt", [(129, 1, 0), (300, 2, 0), (200, 1, 150), (140, 9, 0)])
def test_many_sequences(gpu, n_seq, each, prompt):
    """More sequences than spans are fitted to; a prompt among them; some pause."""
    rng = np.random.default_rng(n_seq)
    new = [0 if i % 7 == 3 else each for i in range(n_seq)]
    lens = [int(n + rng.integers(0, 500)) for n in new]
    lens[5] += 3000
    if prompt:
        new[n_seq // 2], lens[n_seq // 2] = prompt, prompt + 100
    c = Cache(gpu, lens, new, n_head_kv=2, seed=n_seq)
    q = queries(c, 8)
    want, size = attention(c, q)
    close(run_guarded(gpu, c, q, max(lens)), want, size, -(-max(lens) // 64))


def test_long_context_of_few_tokens(gpu):
    """Thousands of positions for 1 to 5 tokens, by every number of rows that a tile has."""
    for new, n_head, n_head_kv in ((1, 24, 4), (2, 24, 4), (5, 24, 4), (4, 32, 1)):
        c = Cache(gpu, [15000], [new], n_head_kv=n_head_kv, seed=new)
        q = queries(c, n_head)
        want, size = attention(c, q)
        close(run_attention(gpu, c, q), want, size, 235)


def test_a_sequence_does_not_change_with_its_neighbours_pages(gpu):
    """A chat's outputs beside a prompt and alone: within the bound of both (the division differs, and with it the last bits)."""
    c = Cache(gpu, [6000, 500], [1, 300], seed=21)
    q = queries(c, 24)
    want, size = attention(c, q)
    out = run_guarded(gpu, c, q, 6000)
    close(out, want, size, 94)
    start = c.view._keep[3]
    start[1:] = 1                                       # the prompt pauses: its rows are nobody's
    alone = run_guarded(gpu, c, q, 6000)
    close(alone[:1], want[:1], size[:1], 94)
    assert bool((alone[1:] == 7).all())


@pytest.mark.parametrize("lens,new,n_head,n_head_kv,scale", [([300], [2], 200, 1, 0.0625), ([300, 90], [5, 3], 200, 1, 0.0625), ([200], [40], 24, 4, -0.0625), ([200], [3], 24, 4, 0.0),
                                                             ([300, 64], [150, 1], 24, 4, 0.0)])
def test_wide_groups_and_other_scales(gpu, lens, new, n_head, n_head_kv, scale):
    """More query heads to a kv head than a tile has rows; scores that are turned round, or all the same."""
    import torch
    c = Cache(gpu, lens, new, n_head_kv=n_head_kv, seed=n_head)
    q = queries(c, n_head)
    want, size = attention(c, q, scale=scale)
    close(run_attention(gpu, c, q, scale=scale), want, size, -(-max(lens) // 64))


def test_two_calls_at_once(gpu):
    """Two caches on two streams, each with its own workspace, run over each other: the bits of each by itself."""
    import torch
    made = []
    for i, (lens, new) in enumerate((([6000, 400], [1, 300]), ([3000, 2000, 900], [2, 2, 90]))):
        c = Cache(gpu, lens, new, seed=30 + i)
        q = queries(c, 24, 40 + i)
        made.append((c, q, run_attention(gpu, c, q), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i, (c, q, _, stream) in enumerate(made):
            with torch.cuda.stream(stream):
                outs[i].append(run_attention(gpu, c, q))
    torch.cuda.synchronize()
    for (_, _, want, _), got in zip(made, outs):
        assert all(torch.equal(want, o) for o in got)
