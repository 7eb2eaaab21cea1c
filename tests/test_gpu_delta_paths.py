"""The delta rule where its kernels take another way: chunks that change between products and single tokens, addresses off 16 bytes, many sequences, replayed calls, rows that
several sequences claim."""
import math

import numpy as np
import pytest

from test_gpu_sequences import DELTA_TOL, delta, delta_inputs, ints, near, run_delta, starts, status_is_clear  # noqa: F401

pytestmark = pytest.mark.gpu


def near_by_parts(got, want, parts):
    """Each range of tokens and each head by its own largest output."""
    for lo, hi in parts:
        err, size = (got[lo:hi].double() - want[lo:hi]).abs().amax((0, 2)), want[lo:hi].abs().amax((0, 2))
        assert bool((err <= DELTA_TOL * size).all()), (lo, hi, (err / size).max().item())


@pytest.mark.parametrize("case", ["value", "steps", "grows"])
@pytest.mark.parametrize("at", [128, 150, 190])
def test_one_chunk_token_by_token(gpu, case, at):
    """A chunk in the middle of a sequence, of one head, holds what sums of products may not; those in front, those behind and the other heads' go on by products."""
    import torch
    n = 330
    q, k, v, g, beta = delta_inputs(n, 1, 3, 128, 128, 17)
    state = torch.randn(1, 3, 128, 128, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    back = at + 2
    if case == "value":                                 # one value past 2^60, forgotten by the next token but one
        v[at, 1] = 1e20
        g[back, 1] = -math.inf
    elif case == "steps":                               # a step past 1e30: the records of the chunk say so
        beta[at, 1] = 2e30
        g[back, 1] = -math.inf
    else:                                               # the state grows by e^50 in one chunk and comes back in the next
        back = 64 * (at // 64 + 1) + 5
        g[at, 1], g[back, 1] = 50.0, -50.0
    want, S = delta(state, q, k, v, g, beta, [0, n], [0])
    assert bool(want.isfinite().all()) and want.abs().max().item() > 1e15
    out = run_delta(gpu, state, (q, k, v, g, beta), [n])
    near_by_parts(out, want, [(0, 64), (64, 128), (128, at), (at, back), (back, 64 * (back // 64 + 1)), (64 * (back // 64 + 1), n)] if at > 128 else
                  [(0, 64), (64, at), (at, back), (back, 64 * (back // 64 + 1)), (64 * (back // 64 + 1), n)])
    for h in range(3):
        near(state[0, h], S[0, h])


@pytest.mark.parametrize("case", ["forgotten", "columns", "zeros"])
def test_values_far_apart_in_a_chunk(gpu, case):
    """2^40 between the values of a chunk, below the 2^60 that leave the products: of tokens behind a large one that is forgotten, of neighbouring columns; zeros are not small values."""
    import torch
    n = 200
    q, k, v, g, beta = delta_inputs(n, 1, 3, 128, 128, 19)
    state = torch.zeros(1, 3, 128, 128, device="cuda")
    cuts = [(0, 64), (64, 128), (128, 192), (192, n)]
    cols = [slice(0, 128)]
    if case == "forgotten":
        v[70, 1] *= 2.0 ** 40
        g[73, 1] = -math.inf
        cuts = [(0, 64), (64, 70), (70, 73), (73, 128), (128, 192), (192, n)]
    elif case == "columns":
        v[:, 1, 17] *= 2.0 ** 40
        cols = [slice(0, 17), slice(17, 18), slice(18, 128)]
    else:
        v[::3] = 0.0
        v[:, :, 5:30] = 0.0
        k[64:70] = 0.0
    want, S = delta(state, q, k, v, g, beta, [0, n], [0])
    out = run_delta(gpu, state, (q, k, v, g, beta), [n])
    for c in cols:
        near_by_parts(out[..., c], want[..., c], cuts)
        for h in range(3):
            near(state[0, h, :, c], S[0, h, :, c])


@pytest.mark.parametrize("new,kh,vh,V", [([1] * 6, 16, 48, 128), ([3, 70, 1], 2, 6, 128), ([200], 1, 2, 128), ([9, 2], 1, 2, 32)])
@pytest.mark.parametrize("off", ["state", "q", "k", "v", "out", "all"])
def test_addresses(gpu, new, kh, vh, V, off):
    """Tensors that begin 4 bytes behind a boundary of 16: each by itself, and all of them."""
    import torch
    n = sum(new)
    args = delta_inputs(n, kh, vh, 128, V, 7)
    state = torch.randn(len(new), vh, 128, V, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda") * 0.1
    want, S = delta(state, *args, starts(new), range(len(new)))

    def moved(x, name):
        if off not in (name, "all"):
            return x
        room = torch.full((x.numel() + 9,), 5.0, device="cuda")
        y = room[1:1 + x.numel()].view(x.shape)
        y.copy_(x)
        return y
    st = moved(state, "state")
    q, k, v, g, beta = (moved(x, name) for x, name in zip(args, ("q", "k", "v", "g", "beta")))
    out = moved(torch.full_like(v, 7.0), "out")
    size = gpu.gdn_seqs_workspace(n, len(new), kh, vh, 128, V)
    ws = torch.full((size // 4,), math.nan, device="cuda") if size else None
    assert gpu.gdn_seqs(st, q, k, v, g, beta, out, ints(starts(new)), None, ws, size, len(new), len(new), n, kh, vh, 128, V) == 0
    near(out, want)
    near(st, S)


@pytest.mark.parametrize("n_seq,each", [(40, 30), (70, 2), (33, 64)])
def test_more_sequences_than_a_warp_has_lanes(gpu, n_seq, each):
    """In chunks and token by token; some pause, some have more."""
    import torch
    new = [0 if i % 9 == 4 else each for i in range(n_seq)]
    new[32], new[n_seq - 1] = 90, 1
    args = delta_inputs(sum(new) + 2, 1, 2, 128, 128, n_seq)
    state = torch.randn(n_seq, 2, 128, 128, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda") * 0.1
    slots = np.random.default_rng(n_seq).permutation(n_seq).tolist()
    want, S = delta(state, *args, starts(new), slots)
    out = run_delta(gpu, state, args, new, slots)
    near(out[:sum(new)], want[:sum(new)])
    near(state, S)
    assert bool((out[sum(new):] == 7).all())


def test_captured_calls_follow_the_numbers(gpu):
    """One graph, replayed with other rows and slots: the bits of the call by itself, whatever goes in chunks."""
    import torch
    n, kh, vh = 160, 2, 6
    args = [x.clone() for x in delta_inputs(n, kh, vh, 128, 128, 9)]
    state, out = torch.zeros(4, vh, 128, 128, device="cuda"), torch.empty(n, vh, 128, device="cuda")
    start, slot = ints([0, 150, 155, 160]), ints([0, 1, 2])
    size = gpu.gdn_seqs_workspace(n, 3, kh, vh, 128, 128)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    step = lambda: gpu.gdn_seqs(state, *args, out, start, slot, ws, size, 3, 4, n, kh, vh, 128, 128)  # noqa: E731
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(st):
        assert step() == 0
        with torch.cuda.graph(graph, stream=st):
            assert step() == 0
    torch.cuda.synchronize()
    first = torch.randn(4, vh, 128, 128, device="cuda") * 0.1
    for new, slots in (([150, 5, 5], [3, 0, 1]), ([1, 1, 1], [1, 3, 2]), ([30, 100, 30], [0, 2, 3]), ([0, 0, 64], [2, 2, 1]), ([0, 0, 0], [0, 0, 0])):
        start.copy_(ints(starts(new)))
        slot.copy_(ints(slots))
        for x in args[:3]:
            x.copy_(x.roll(1, 0))
        want, S = delta(first, *args, starts(new), slots)
        got = []
        for go in (graph.replay, step):
            state.copy_(first)
            out.fill_(7.0)
            torch.cuda.synchronize()
            assert not go()
            torch.cuda.synchronize()
            got.append((out.clone(), state.clone()))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
        m = sum(new)
        assert bool((out[m:] == 7).all())
        if m:
            near(out[:m], want[:m])
            near(state, S)
        else:
            assert torch.equal(state, first)


@pytest.mark.parametrize("first,last", [(200, 200), (200, 20), (24, 200)])
def test_rows_that_several_sequences_claim(gpu, first, last):
    """Of three sequences the second's rows run backwards and the others claim the same ones: the status word says so, the second keeps its state, and nothing outside the call's
    memory is written."""
    import torch
    n, kh, vh = 200, 2, 6
    args = delta_inputs(n, kh, vh, 128, 128, 3)
    state = torch.randn(3, vh, 128, 128, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda") * 0.1

    def guarded(x):
        room = torch.full((x.numel() + 2048,), 3.0, device="cuda")
        y = room[1024:1024 + x.numel()].view(x.shape)
        y.copy_(x)
        return room, y
    state_room, st = guarded(state)
    out_room, out = guarded(torch.full((n, vh, 128), 7.0, device="cuda"))
    size = gpu.gdn_seqs_workspace(n, 3, kh, vh, 128, 128)
    ws_room, ws = guarded(torch.full((size // 4,), 1.0, device="cuda"))
    assert gpu.gdn_seqs(st, *args, out, ints([0, first, 0, last]), None, ws, size, 3, 3, n, kh, vh, 128, 128) == 0
    assert gpu.device_status() == 3 and gpu.clear_status() == 0
    for room in (state_room, out_room, ws_room):
        assert bool((room[:1024] == 3).all()) and bool((room[-1024:] == 3).all())
    assert torch.equal(st[1], state[1])
    # the first sequence is served; what the last one makes of its rows is not said, where it is served at all
    want, S = delta(state, *args, [0, first], [0])
    near(st[0], S[0])
    assert bool((out[max(first, last):] == 7).all()) and bool(out.isfinite().all())
