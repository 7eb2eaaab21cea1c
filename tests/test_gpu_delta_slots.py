"""Slots of the delta rule's states: who may name which."""
import pytest

from test_gpu_sequences import delta, delta_inputs, near, run_delta, starts, status_is_clear  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [[3, 0, 2, 0], [0, 70, 130, 0], [40, 0, 1, 0]])
def test_slots_of_sequences_without_tokens(gpu, new):
    """A call with room for four sequences, two of them without new tokens: the slots of those may be anybody's, or none of the pool, and stop nobody."""
    import torch
    args = delta_inputs(sum(new), 2, 6, 128, 128, 3)
    first = torch.randn(5, 6, 128, 128, device="cuda") * 0.1
    busy = [s for s in range(4) if new[s]]
    for spare in (4, 1, -1, 5, 2 ** 31 - 1):
        slots = [spare] * 4
        slots[busy[0]], slots[busy[1]] = 4, 1
        state = first.clone()
        want, S = delta(state, *args, starts(new), [x if n else 0 for x, n in zip(slots, new)])
        out = run_delta(gpu, state, args, new, slots)
        assert gpu.device_status() == 0
        near(out, want)
        near(state, S)
        for s in (0, 2, 3):
            assert torch.equal(state[s], first[s])


@pytest.mark.parametrize("new", [[1] * 4, [2, 1, 1, 30], [70, 2, 1, 1]])
def test_slots_of_many_columns(gpu, new):
    """48 heads: a CTA has 128 columns of a state.  Slots in any order; two that are the same stop both of their sequences and no other."""
    import torch
    args = delta_inputs(sum(new), 16, 48, 128, 128, 5)
    first = torch.randn(6, 48, 128, 128, device="cuda") * 0.1
    state = first.clone()
    want, S = delta(state, *args, starts(new), [5, 0, 3, 1])
    out = run_delta(gpu, state, args, new, [5, 0, 3, 1])
    near(out, want)
    near(state, S)
    state.copy_(first)
    out = run_delta(gpu, state, args, new, [5, 0, 3, 5])
    assert gpu.device_status() == 3 and gpu.clear_status() == 0
    lo, hi = new[0], new[0] + new[1] + new[2]
    near(out[lo:hi], want[lo:hi])
    assert bool((out[:lo] == 7).all()) and bool((out[hi:] == 7).all())
    for s in (0, 3):
        near(state[s], S[s])
    for s in (1, 2, 4, 5):
        assert torch.equal(state[s], first[s])
