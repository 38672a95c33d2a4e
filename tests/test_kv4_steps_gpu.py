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


def test_lengths_carried_on(fn, kv4):
    """step.ctx: the new length of a served request, the old one of a refused or idle one, 0 of a finished one."""
    table = torch.full((6, 3), -1, dtype=torch.int32, device="cuda")
    table[0, :2], table[1, :1], table[3, :2], table[4, :1] = i32(0, 1), i32(2), i32(3, 4), i32(5)
    free = torch.zeros(8, dtype=torch.int32, device="cuda")
    free[:1] = 6
    # served within its page; one page taken; none left; finished (its pages come too late for none: they are pushed first); idle; too long
    ctx, add = i32(20, 16, -3, 32, 7, 0), i32(5, 1, 0, 1, 0, 49)
    for room in (64, 5000):  # rows written by the planning kernel, and by the one after it
        t, f = table.clone(), free.clone()
        step = kv4.KV4Planner(fn, 16).plan(ctx, add, t, f, i32(1), room)
        assert step.ctx.tolist() == [25, 17, 0, 32, 7, 0] and step.kv_len.tolist() == [25, 17, 0, 0, 7, 0]
        assert int(step.status) == 2 and int(step.free_count) == 0
        step = kv4.KV4Planner(fn, 16).plan(ctx, i32(-1, 0, 0, 1, -1, 1), table.clone(), free.clone(), i32(1), room)
        assert step.ctx.tolist() == [0, 16, 0, 33, 0, 1] and int(step.status) == 0


def test_the_documented_loop_survives_a_shortage(fn, kv4):
    """Steps as the module's documentation writes them, with too few pages at times: a refused request goes on later where it stood, and
    no page is lost or in two places."""
    rng = np.random.default_rng(1)
    n, bs, width, n_pages, room = 5, 16, 6, 11, 64
    planner = kv4.KV4Planner(fn, bs)
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    free = torch.arange(n_pages, dtype=torch.int32, device="cuda")
    ctx, free_count = torch.zeros(n, dtype=torch.int32, device="cuda"), i32(n_pages)
    refused, length = 0, np.zeros(n, np.int64)
    for _ in range(200):
        add = np.where(length == 0, rng.integers(0, 30, n), rng.integers(0, 4, n))
        add[(rng.random(n) < 0.08) | (length + add > width * bs)] = -1
        step = planner.plan(ctx, i32(*add.tolist()), table, free, free_count, max_tokens=room)
        ctx.copy_(step.ctx)
        free_count.copy_(step.free_count)
        served = step.kv_len.cpu().numpy() > 0
        refused += int(step.status)
        length = np.where(add < 0, 0, np.where((add > 0) & ~served, length, length + add))
        assert ctx.tolist() == length.tolist()
        held = [int(p) for r in range(n) for p in table[r, :-(-int(length[r]) // bs)].tolist()]
        ids = free[:int(free_count)].tolist() + held
        assert sorted(ids) == list(range(n_pages))
    assert refused > 10 and length.sum() > 0


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
