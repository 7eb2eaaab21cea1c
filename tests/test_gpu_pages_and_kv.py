"""The cache in pages beside the cache of one sequence (include/bonsai_kv.h), which it is defined by.

Both store Q8_0 rows.  One takes a block's scale as its largest magnitude over 127, the other as its product with 1 / 127: the fp32 scales differ in the last bit in one block of
21, the fp16 ones that are stored in none (every fp32 magnitude looked at), a code whose quotient lies beside a half in one value of 10^7, by one.
"""
import numpy as np
import pytest

from test_gpu_sequences import Cache, ints, status_is_clear  # noqa: F401

pytestmark = pytest.mark.gpu
H, HKV, D = 24, 4, 256


def kv_rows(gpu, kv, layer, cap, n):
    """K and V rows of one layer as bytes: [2][heads][n][8][34]."""
    import torch
    kp, vp, size = kv.arrays()

    def raw(ptr):
        class Raw:
            __cuda_array_interface__ = {"shape": (size,), "typestr": "|u1", "data": (int(ptr), False), "version": 3}
        return torch.as_tensor(Raw(), device="cuda").cpu().numpy().reshape(16, HKV, cap, 8, 34)[layer, :, :n]
    return np.stack([raw(kp), raw(vp)])


def page_rows(c, s, n):
    """The same of sequence s of a paged cache of one layer."""
    pool = c.d_pool.cpu().numpy()[c.table[s, :-(-n // 64)], 0]              # pages, K | V, heads, positions, blocks, bytes
    return pool.transpose(1, 2, 0, 3, 4, 5).reshape(2, HKV, -1, 8, 34)[:, :, :n]


def whole_scales(x):
    """Every block's largest magnitude 127 times a power of two: product and quotient are the same scale."""
    import torch
    b = x.reshape(*x.shape[:-1], -1, 32).clone()
    top = torch.exp2(torch.ceil(torch.log2(b.abs().amax(-1, keepdim=True))) - 6)
    b[..., :1] = 127 * top / 64
    b[..., 1:] = b[..., 1:].clamp(-1.9 * top, 1.9 * top)
    return b.reshape(x.shape)


@pytest.mark.parametrize("whole", [False, True])
def test_rows(gpu, whole):
    import torch
    n, layer = 700, 3
    g = torch.Generator(device="cuda").manual_seed(41)
    k, v = (torch.randn(n, HKV, D, generator=g, device="cuda") * torch.exp(2 * torch.randn(n, HKV, 1, generator=g, device="cuda")) for _ in range(2))
    if whole:
        k, v = whole_scales(k), whole_scales(v)
    kv = gpu.KVCache(n + 5)
    assert kv.append_batch(layer, 0, n, k, v) == 0
    c = Cache(gpu, [n], [n])
    assert c.view.append(0, k, v) == 0
    one, paged = kv_rows(gpu, kv, layer, n + 5, n), page_rows(c, 0, n)
    kv.close()
    assert np.array_equal(one[..., :2], paged[..., :2])
    off = np.abs(one[..., 2:].view(np.int8).astype(int) - paged[..., 2:].view(np.int8))
    # 1.4 million codes: 0.17 of them differ on average, and not by more than one
    assert off.max() <= 1 and off.sum() <= (0 if whole else 6)


@pytest.mark.parametrize("n,new", [(1, 1), (700, 1), (700, 3), (2000, 21), (300, 300)])
def test_attention(gpu, n, new):
    """Equal caches and queries: each new token's outputs are those of bonsai_kv_attn_decode at its position, by every kernel that serves such a number of tokens."""
    import torch
    layer = 5
    g = torch.Generator(device="cuda").manual_seed(n + new)
    k, v = (whole_scales(torch.randn(n, HKV, D, generator=g, device="cuda")) for _ in range(2))
    q = whole_scales(torch.randn(new, H, D, generator=g, device="cuda"))
    kv = gpu.KVCache(n)
    assert kv.append_batch(layer, 0, n, k, v) == 0
    c = Cache(gpu, [n, 40], [n, 0])
    assert c.view.append(0, k, v) == 0
    view = gpu.Pages(c.d_pool, ints(c.table), ints([n, 40]), ints([0, new, new]), 1, HKV, new)
    size = view.attn_workspace(n, H)
    out, want = torch.empty_like(q), torch.empty_like(q)
    assert view.attn(0, q, out, H, n, torch.empty(size, dtype=torch.uint8, device="cuda") if size else None, 0.0625) == 0
    for t in range(new):
        assert kv.attn_decode(layer, n - new + t, q[t], want[t]) == 0
    torch.cuda.synchronize()
    kv.close()
    # each side is within 1e-5 of the largest output of the value (as its own tests have it)
    err = (out - want).abs().amax((1, 2)) / want.abs().amax((1, 2))
    assert err.max().item() <= 2e-5


@pytest.mark.parametrize("new", [1, 3, 40, 130])
def test_queries_that_are_no_numbers(gpu, new):
    """An infinity or NaN in a query is its own row's: what bonsai_kv_attn_decode makes of it, and nothing of any other row's."""
    import torch
    n, layer = 400, 2
    g = torch.Generator(device="cuda").manual_seed(new)
    k, v = (whole_scales(torch.randn(n, HKV, D, generator=g, device="cuda")) for _ in range(2))
    q = whole_scales(torch.randn(new, H, D, generator=g, device="cuda"))
    q[new // 2, 3, 40], q[new // 2, 9, 0], q[new - 1, 23, 255] = float("inf"), float("nan"), float("-inf")
    kv = gpu.KVCache(n)
    assert kv.append_batch(layer, 0, n, k, v) == 0
    c = Cache(gpu, [n], [n])
    assert c.view.append(0, k, v) == 0
    view = gpu.Pages(c.d_pool, ints(c.table), ints([n]), ints([0, new]), 1, HKV, new)
    size = view.attn_workspace(n, H)
    out, want = torch.empty_like(q), torch.empty_like(q)
    assert view.attn(0, q, out, H, n, torch.empty(size, dtype=torch.uint8, device="cuda") if size else None, 0.0625) == 0
    for t in range(new):
        assert kv.attn_decode(layer, n - new + t, q[t], want[t]) == 0
    torch.cuda.synchronize()
    kv.close()
    odd = [(new // 2, 3), (new - 1, 23)]
    for t, h in odd:
        assert bool((~out[t, h].isfinite()).all()) and bool((~want[t, h].isfinite()).all())
        out[t, h] = want[t, h] = 0.0
    assert bool(out.isfinite().all())
    assert ((out - want).abs().amax((1, 2)) / want.abs().amax((1, 2))).max().item() <= 2e-5
