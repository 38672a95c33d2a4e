"""CPU: an object whose calls pass pointers that were taken once keeps the tensors they are of."""

import pytest
import torch


def test_a_weight_keeps_its_tensors():
    from fp8 import CODES, Fp8Weight
    w = Fp8Weight.__new__(Fp8Weight)
    w._keep(None, torch.zeros(3, 64).to(CODES), torch.ones(1, 1))
    q, scale = w.q, w.scale
    for name, other in (("q", q.clone()), ("scale", scale.clone()), ("rows", 2), ("cols", 48)):
        with pytest.raises(AttributeError, match=name):
            setattr(w, name, other)
    assert w.q is q and w.scale is scale and (w.rows, w.cols) == (3, 64)
    w.scale.fill_(2)
    assert (w.values() == 0).all() and w.values().shape == (3, 64)


def test_a_plan_a_workspace_and_a_cache_keep_theirs():
    from kv4 import KV4Cache, KV4Plan, KV4Workspace
    plan = KV4Plan(2, 3, "cpu")
    for name in ("cu", "kv_len", "ctx", "slots", "positions", "requests", "free_count", "status"):
        with pytest.raises(AttributeError, match=name):
            setattr(plan, name, getattr(plan, name).clone())
    assert plan.ptrs == [t.data_ptr() for t in (plan.cu, plan.kv_len, plan.slots, plan.positions, plan.requests, plan.status, plan.ctx)]
    ws = KV4Workspace(type("Fn", (), {"kv4_attn_workspace": lambda self: 64})(), "cpu")
    cache = KV4Cache.__new__(KV4Cache)
    cache.pages = torch.zeros(4, dtype=torch.uint8)
    for o, name in ((ws, "tensor"), (cache, "pages")):
        with pytest.raises(AttributeError, match=name):
            setattr(o, name, getattr(o, name).clone())
    assert ws.ptr == ws.tensor.data_ptr()
