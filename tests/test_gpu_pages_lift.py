"""Attention over shared pages where scores are sums of few products, which the tensor core does not cut off: what such scores are lifted by all the same moves outputs by no more than is stated."""
import math

import numpy as np
import pytest

from test_gpu_pages_division import attention as plain_attention
from test_gpu_pages_shared import FORMS, cache_of, close, run
from test_gpu_sequences import U, status_is_clear  # noqa: F401

pytestmark = pytest.mark.gpu
LIFT = 6 * 2.0 ** -23


def bound(c, size):
    """Scores times 1 + LIFT move an output by LIFT times the covariance of scores and values under the weights: at most the largest standard deviation that n scores have under their own weights,
    sqrt(ln(n)^2 / 4 + 1), times the largest |v|.  Roundings, in u of size: a score's planes without low times low 4, three sums of one product each 6, factors 5, less its reference 2; a weight
    9; an output's planes 4, 24 matrix instructions 48, and 3 a page, the sum of weights 3 a page, division and product 3 each.  Weights are multiples of 2^-32 of a row's largest."""
    n = max(c.lens)
    most_v = max(np.abs(c.rows(s, 0, 1, j)).max() for s, m in enumerate(c.lens) if m for j in range(c.hkv))
    return size * U * (17 + 9 + 52 + 6 + 6 * -(-n // 64)) + most_v * (LIFT * math.sqrt(math.log(n) ** 2 / 4 + 1) + n * 2.0 ** -32)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("scale", [0.01, 0.0625, 0.3, 1.0])
@pytest.mark.parametrize("values", ["random", "two camps"])
def test_scores_of_one_product(gpu, form, scale, values):
    """Queries with one value that is not zero, of either sign, in any dim."""
    import torch
    c = cache_of(gpu, form)
    if values == "two camps":           # v is 1 where the first of k's codes is positive, else -1: the values that a change of scores moves most
        k, v = c.pool[:, 0, 0].reshape(-1, 8, 34), c.pool[:, 0, 1].copy().reshape(-1, 8, 34)
        v[..., :2] = np.array([1 / 127], np.float16).view(np.uint8)
        v[..., 2:] = np.where(k[:, :1, 2:3].view(np.int8) > 0, 127, -127).astype(np.int8).view(np.uint8)
        c.pool[:, 0, 1] = v.reshape(c.pool[:, 0, 1].shape)
        c.upload()
    g = torch.Generator(device="cuda").manual_seed(7)
    q = torch.zeros(c.n_tok, 24, 256, device="cuda")
    dim = torch.randint(0, 256, (c.n_tok, 24, 1), generator=g, device="cuda") if values == "random" else torch.zeros(c.n_tok, 24, 1, dtype=torch.int64, device="cuda")
    q.scatter_(-1, dim, 4 * torch.randn(c.n_tok, 24, 1, generator=g, device="cuda"))
    want, size = plain_attention(c, q, scale=scale)
    close(run(c, q, scale=scale), want, bound(c, size))
