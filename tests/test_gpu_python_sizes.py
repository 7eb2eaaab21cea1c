"""The calls for several sequences refuse a tensor that is smaller than the sizes beside it say; tensors that hold them exactly are served."""
import pytest

pytestmark = pytest.mark.gpu


def each_too_small(call, tensors, names):
    """tensors: flat ones of exactly the size that the call needs.  call(list of tensors) -> rc."""
    assert call(tensors) == 0
    for i, name in enumerate(names):
        short = list(tensors)
        short[i] = tensors[i][:-1]
        if short[i].storage_offset() + short[i].numel() < short[i].untyped_storage().nbytes() // short[i].element_size():
            short[i] = short[i].clone()                 # (a strided input may go to the end of its memory)
        with pytest.raises(RuntimeError, match=f"{name} is smaller than the sizes"):
            call(short)


@pytest.mark.parametrize("n_head,n_head_kv,dim,n_rot,gate", [(3, 1, 64, 32, False), (4, 2, 256, 64, True), (1, 1, 33, 2, False)])
def test_head_norms(gpu, n_head, n_head_kv, dim, n_rot, gate):
    import torch
    n, wide = 5, 2 * dim if gate else dim
    t = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    last = lambda heads: (n * heads - 1) * wide + dim  # noqa: E731  (the last row's gate need not be there)
    tensors = [t(last(n_head)), t(last(n_head_kv)), t(dim), t(dim), t(n, dtype=torch.int32), t(n_rot // 2, dtype=torch.float64), t(n * n_head * dim), t(n * n_head_kv * dim)]
    each_too_small(lambda x: gpu.qk_norm_rope(*x, n, n_head, n_head_kv, dim, n_rot, n_head * wide, wide, n_head_kv * wide, wide, 1e-6), tensors,
                   ["q", "k", "q_weight", "k_weight", "pos", "freq", "q_out", "k_out"])
    # what is not read need not be there
    none = torch.empty(0, device="cuda")
    x = list(tensors)
    x[1] = x[3] = x[7] = none
    assert gpu.qk_norm_rope(*x, n, n_head, 0, dim, n_rot, n_head * wide, wide, 0, 0, 1e-6) == 0
    x[4] = x[5] = None
    assert gpu.qk_norm_rope(*x, n, n_head, 0, dim, 0, n_head * wide, wide, 0, 0, 1e-6) == 0


def test_pages(gpu):
    import torch
    hkv, h, n = 2, 6, 3
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    pool = torch.zeros(9, 2 * hkv * 64 * 272, dtype=torch.uint8, device="cuda")
    view = gpu.Pages(pool, i32([[0, 1, 2, 3, 4, 5]]), i32([300]), i32([0, n]), 1, hkv, n)
    rows = lambda heads: torch.zeros(n * heads * 256, device="cuda")  # noqa: E731
    each_too_small(lambda x: view.append(0, *x), [rows(hkv), rows(hkv)], ["k", "v"])
    size = view.attn_workspace(300, h)
    assert size > 0
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
    each_too_small(lambda x: view.attn(0, *x, h, 300, ws, 0.0625), [rows(h), rows(h)], ["q", "out"])
    call = gpu._native().pages_attn
    each_too_small(lambda x: call(view._struct(), 0, rows(h), rows(h), h, 300, x[0], size, 0.0625), [ws], ["workspace"])
    src, dst = torch.tensor([0], dtype=torch.int32), torch.tensor([8], dtype=torch.int32)
    each_too_small(lambda x: gpu.pages_copy(x[0], pool.shape[1], 9, src, dst, 1), [pool.flatten()], ["pool"])
    assert gpu.pages_copy(pool, pool.shape[1], 9, src, dst, 0) == 0


def test_delta(gpu):
    import torch
    n, kh, vh, seqs, slots = 70, 1, 2, 2, 3
    t = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    size = gpu.gdn_seqs_workspace(n, seqs, kh, vh, 128, 128)
    assert size > 0
    start, slot = torch.tensor([0, 68, 70], dtype=torch.int32, device="cuda"), torch.tensor([2, 0], dtype=torch.int32, device="cuda")
    tensors = [t(slots * vh * 128 * 128), t(n * kh * 128), t(n * kh * 128), t(n * vh * 128), t(n * vh), t(n * vh), t(n * vh * 128), start, slot, t(size, dtype=torch.uint8)]
    each_too_small(lambda x: gpu.gdn_seqs(*x, size, seqs, slots, n, kh, vh, 128, 128), tensors,
                   ["state", "q", "k", "v", "g", "beta", "out", "start", "slot", "workspace"])
    x = list(tensors)
    x[8] = None
    assert gpu.gdn_seqs(*x, size, seqs, slots, n, kh, vh, 128, 128) == 0
    assert gpu.device_status() == 0
