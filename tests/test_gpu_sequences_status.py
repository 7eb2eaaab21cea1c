"""What the status word says when more than one thing went wrong."""
import pytest

from test_gpu_sequences import Cache, ints

pytestmark = pytest.mark.gpu


def run_out(gpu):
    """A two-rank list of which one rank never comes: the wait for it ends after 3 ms, and the status word says so."""
    import torch
    from bonsai_b200 import synth
    payload = 4096

    class TwoBuffers:
        rank, world, counter_offset, total_bytes = 0, 2, payload, payload + 64
    mine, nobody = (torch.zeros(payload + 64, dtype=torch.uint8, device="cuda") for _ in range(2))
    TwoBuffers.ptrs = [mine.data_ptr(), nobody.data_ptr()]
    W = torch.from_numpy(synth.pq2_0_weights(64, 1024, seed=5)).cuda()
    x = torch.from_numpy(synth.activations(1024, seed=5)).cuda()
    chain = gpu.Chain([(W, x, None, mine[:256].view(torch.float32), 64, 1024, gpu.OP_ROTATE)], peers=TwoBuffers, wait_limit_us=3000)
    assert chain.run() == 0
    torch.cuda.synchronize()
    chain.close()


def test_a_wait_that_ran_out_stays_reported(gpu):
    """Numbers that do not fit come after it: the wait's report is not lost.  Once it is cleared, theirs is the next."""
    import torch
    c = Cache(gpu, [300, 200], [2, 2], seed=10)
    k = torch.randn(c.n_tok, 4, 256, device="cuda")
    c.view._keep[1][1, 3] = c.n_pages                   # a page that the pool does not have
    try:
        assert gpu.device_status() == 0
        run_out(gpu)
        assert gpu.device_status() == 2
        assert c.view.append(0, k, k) == 0
        assert gpu.device_status() == 2 and gpu.clear_status() == 0
        assert c.view.append(0, k, k) == 0
        assert gpu.device_status() == 3
        c.view._keep[1].copy_(ints(c.table))
        assert c.view.append(0, k, k) == 0
        assert gpu.device_status() == 3 and gpu.clear_status() == 0
        assert c.view.append(0, k, k) == 0
        assert gpu.device_status() == 0
    finally:
        gpu.clear_status()
