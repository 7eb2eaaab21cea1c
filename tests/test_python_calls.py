"""The native calls take what the ctypes calls took: tensors that share memory until they are written, objects with a tensor's
is_cuda, is_contiguous() and data_ptr(); and refuse the rest."""
import pytest


class Like:
    def __init__(self, t=None, cuda=True, contiguous=True):
        self.t, self.is_cuda, self.contiguous = t, cuda, contiguous

    def is_contiguous(self):
        return self.contiguous

    def data_ptr(self):
        return self.t.data_ptr()


def test_refusals():
    import bonsai_b200
    with pytest.raises(RuntimeError, match="no CPU path"):
        bonsai_b200.fwht(Like(cuda=False), None, 1024)
    with pytest.raises(RuntimeError, match="contiguous"):
        bonsai_b200.fwht(Like(contiguous=False), None, 1024)
    with pytest.raises(AttributeError):
        bonsai_b200.fwht(3, None, 1024)


@pytest.mark.gpu
def test_memory_shared_until_written(gpu):
    """An output that is a lazy clone gets memory of its own; what it was cloned from keeps its values."""
    import torch
    x = torch.randn(1024, device="cuda")
    base = torch.full((1024,), 5.0, device="cuda")
    out, want = torch._lazy_clone(base), torch.empty(1024, device="cuda")
    assert gpu.fwht_quant(x, None, None, want, 1024) == 0
    assert gpu.fwht_quant(x, None, None, out, 1024) == 0
    assert bool((base == 5.0).all()) and torch.equal(out, want)
    assert gpu.rmsnorm(torch._lazy_clone(x), base, out, 1, 1024, 1e-6) == 0


@pytest.mark.gpu
def test_objects_like_tensors(gpu):
    import torch
    x = torch.randn(2048, device="cuda")
    y = x.clone()
    assert gpu.fwht(x, None, 2048) == 0 and gpu.fwht(Like(y), None, 2048) == 0
    assert torch.equal(x, y)


NORMS = ["q", "k", "q_weight", "k_weight", "pos", "freq", "q_out", "k_out"]
NORM_SIZES = (1, 1, 1, 64, 2, 64, 64, 64, 64, 1e-6)
DELTA = ["state", "q", "k", "v", "g", "beta", "out", "start", "slot"]
DELTA_SIZES = (None, 0, 1, 1, 1, 1, 1, 32, 32)


def wrong(names, own):
    """(which argument, a type that it is not read as): every argument of a call and the likeliest mistakes."""
    import torch
    for i, name in enumerate(names):
        for t in (torch.int64, torch.int32, torch.float64, torch.float32, torch.bfloat16, torch.uint8):
            if t != own.get(name, torch.float32):
                yield i, name, torch.zeros(64, dtype=t)


def test_types_that_are_not_read():
    """A tensor of another type than the call reads is refused, wherever it lies: torch's default int64 is not read as int32, nor float32 as double."""
    import torch
    import bonsai_b200 as bb
    for i, name, t in wrong(NORMS, {"pos": torch.int32, "freq": torch.float64}):
        args = [None] * 8
        args[i] = t
        with pytest.raises(RuntimeError, match=f"^{name} must be a tensor of"):
            bb.qk_norm_rope(*args, *NORM_SIZES)
    for i, name, t in wrong(DELTA, {"start": torch.int32, "slot": torch.int32}):
        args = [None] * 9
        args[i] = t
        with pytest.raises(RuntimeError, match=f"^{name} must be a tensor of"):
            bb.gdn_seqs(*args, *DELTA_SIZES)
    calls = bb._native()
    for i, name, t in wrong(["k", "v"], {}):
        with pytest.raises(RuntimeError, match=f"^{name} must be a tensor of"):
            calls.pages_append(None, 0, *((t, None) if i == 0 else (None, t)))
    for i, name, t in wrong(["q", "out"], {}):
        with pytest.raises(RuntimeError, match=f"^{name} must be a tensor of"):
            calls.pages_attn(None, 0, *((t, None) if i == 0 else (None, t)), 24, 100, None, 0, 1.0)
