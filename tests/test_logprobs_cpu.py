"""CPU: the oracle of the token scores against other ways to the same numbers, and the C entry's refusals (before any device work)."""

import numpy as np
import pytest
import torch

from fn import FN
from oracle import logprobs as O


def test_oracle_is_log_softmax():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((20, 37)) * 4
    token = rng.integers(0, 37, 20)
    got = O.rows(x, token, 5)
    want = torch.log_softmax(torch.from_numpy(x), 1).numpy()
    assert np.abs(got["logprob"] - want[np.arange(20), token]).max() < 1e-12
    assert np.abs(got["entropy"] + (np.exp(want) * want).sum(1)).max() < 1e-12
    for r in range(20):
        order = sorted(range(37), key=lambda i: (-x[r, i], i))
        assert list(got["top_ids"][r]) == order[:5]
        assert got["rank"][r] == order.index(token[r])
        assert np.abs(got["top_logprobs"][r] - want[r, order[:5]]).max() < 1e-12


def test_oracle_ties_and_masks():
    x = np.array([1.0, -np.inf, 1.0, 0.0, -0.0, 1.0])
    logprob, rank, entropy, ids, logs = O.row(x, 4, 8)
    assert list(ids) == [0, 2, 5, 3, 4, -1, -1, -1] and rank == 4
    assert (logs[5:] == -np.inf).all() and logs[0] == logs[2]
    assert O.row(x, 1, 0)[0] == -np.inf and O.row(x, 1, 0)[1] == 5
    for i in range(6):
        assert O.row(x, i, 0)[1] == sum(O.before(x, j, i) for j in range(6))
    none = np.full(4, -np.inf)
    logprob, rank, entropy, ids, logs = O.row(none, 2, 2)
    assert logprob == -np.inf and rank == 2 and entropy == 0 and list(ids) == [-1, -1]
    assert O.row(none, -1, 0)[:2] == (0.0, -1)
    sick = np.array([0.0, np.nan, 2.0])
    logprob, rank, entropy, ids, logs = O.row(sick, 1, 3)
    assert np.isnan(logprob) and rank == -1 and np.isnan(entropy) and list(ids) == [2, 0, -1]
    assert O.row(sick, 0, 0)[1] == 1


GOOD = dict(dtype=0, logits=4096, stride=10, rows=2, vocab=10, tokens=4096, logprob=4096, rank=4096, entropy=4096, top=3, top_ids=4096,
            top_logprobs=4096)


@pytest.mark.parametrize("change, words", [
    (dict(dtype=1), "F32 or BF16"), (dict(dtype=12), "F32 or BF16"), (dict(rows=-1), "bad row"), (dict(vocab=0), "bad row"),
    (dict(vocab=(1 << 28) + 1), "bad row"), (dict(top=-1), "top out of range"), (dict(top=33), "top out of range"),
    (dict(logits=None), "null pointer"), (dict(top_ids=None), "null pointer"), (dict(top_logprobs=None), "null pointer"),
    (dict(tokens=None), "want tokens"), (dict(tokens=None, rank=None), "want tokens"), (dict(logits=4098), "aligned"),
    (dict(logits=4097, dtype=30), "aligned")])
def test_refusals(libpath, change, words):
    with pytest.raises(RuntimeError, match=words):
        FN(libpath).logprobs(**{**GOOD, **change})


def test_no_rows_is_no_work(libpath):
    FN(libpath).logprobs(**{**GOOD, "rows": 0})


def test_layer_refuses(libpath):
    from logprobs import token_logprobs
    fn = FN(libpath)
    for bad in (torch.zeros(2, 4), torch.zeros(4), torch.zeros(2, 4, dtype=torch.float16)):
        with pytest.raises(ValueError, match="logits"):
            token_logprobs(fn, bad)
