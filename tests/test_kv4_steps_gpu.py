"""GPU: steps of the paged 4-bit cache one after the other: lengths carried on, refused requests, bounds on the new tokens."""

import numpy as np
import pytest
import torch

from oracle import kv4 as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv4(fn):
    import kv4 as m
    return m


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group, max_new, new", [(8, 7, 14), (8, 1, 30), (2, 5, 19), (8, 0, 6)])
def test_too_small_a_bound_is_not_wrong(fn, kv4, group, max_new, new, dtype):
    """A request of two 64-token tiles with more rows than max_new says."""
    rng = np.random.default_rng(2)
    c = kv4.KV4Cache(fn, 1, 64, 64, 2)
    k, v = (torch.from_numpy(rng.standard_normal((100, 1, 64)).astype(np.float32)).cuda() for _ in range(2))
    c.store(k, v, torch.arange(100, device="cuda"))
    q = torch.from_numpy(rng.standard_normal((new, group, 64)).astype(np.float32)).cuda().to(dtype)
    a = (i32(0, new), i32(100), i32(0, 1)[None])
    got = c.attn(q, *a, max_new=max_new).float().cpu().numpy()
    want = O.attn(c.pages.cpu().numpy(), 64, 64, q.float().cpu().numpy(), [0, new], [100], np.array([[0, 1]]))
    tol = 2e-5 * 4 if dtype == torch.float32 else np.abs(want) * 2.0 ** -8 + 4 * 2.0 ** -10  # as in tests/test_kv4_gpu.py
    assert (np.abs(got - want) <= tol).all()
