"""GPU: requests of different lengths through ServeModel (flashnext/serve.py: planning, norm + RoPE rows, 4-bit store and
attention, DeltaNet places reused) against the float64 oracle, and its new kernels.

The oracle attends over the keys and values that the model stored (read back from its pages): rounding to 4 bits is a step, and
a value that the tensor-core projections' 1e-4 carries over a boundary would differ by all of it. Each stored value is within
one step of the oracle's own; then the batched model's tolerance holds (tests/test_batch_gpu.py): log-probabilities within
1e-3, greedy ids equal where the oracle's top two are more than 1e-2 apart.
"""

import numpy as np
import pytest

from oracle.model import OracleModel, rmsnorm, rope
from synth import model_config, model_weights, rope_inv_freq

pytestmark = pytest.mark.gpu
LOGPROB_TOL, TIE = 1e-3, 1e-2


class Stored(list):
    """An oracle's cache list that keeps what the device stored, after a look that it is the same value."""

    def __init__(self, device):
        super().__init__()
        self.device = device

    def append(self, x):
        got = self.device[len(self)]
        step = np.abs(x.reshape(-1, 64)).max(-1) / 8  # half a step, one at the clipped end, and the scale's rounding
        assert (np.abs(got - x).reshape(-1, 64) <= step[:, None] * 1.01).all()
        super().append(got)


class Kv4Oracle(OracleModel):
    def attend_over(self, stored):
        """stored: per attention layer, ([k per token], [v per token])."""
        self.reset()
        for st, (k, v) in zip((st for st in self.state if "K" in st), stored):
            st["K"], st["V"] = Stored(k), Stored(v)


def logprobs(x):
    x = np.asarray(x, np.float64)
    return x - x.max() - np.log(np.exp(x - x.max()).sum())


@pytest.fixture(scope="module")
def small():
    cfg = model_config(small=True)
    return cfg, model_weights(cfg, 3)


@pytest.fixture(scope="module")
def model(fn, small):
    import torch
    from serve import ServeModel
    m = ServeModel(fn, *small, batch=3, pages=8, max_ctx=48, page_size=16)
    s = torch.cuda.Stream()
    m.capture(s)
    yield m, s
    m.free()


def test_requests_of_different_lengths_match_the_oracle(model, small):
    """Seven requests through three places: admitted as others finish, over page ends, pages reused."""
    m, s = model
    cfg, W = small
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, cfg["vocab"], n) for n in (5, 17, 1, 9, 16, 3, 30)]
    n_new = [12, 4, 20, 1, 8, 15, 3]
    rows, stored = {}, {}
    layers = [L for L in m.layers if L["kind"] != "G"]

    def look(r, at, row):
        b = (row.data_ptr() - m.logits.data_ptr()) // (4 * cfg["vocab"])
        rows.setdefault(r, []).append(row.cpu().numpy().copy())
        for i, L in enumerate(layers):
            k, v = L["cache"].load(m.plan.slots[b:b + 1])
            st = stored.setdefault(r, [([], []) for _ in layers])[i]
            st[0].append(k[0].cpu().numpy().astype(np.float64))
            st[1].append(v[0].cpu().numpy().astype(np.float64))

    outs = m.generate(prompts, n_new, s, logits=look)
    oracle, worst = Kv4Oracle(cfg, W, rope_inv_freq(cfg["rope_base"])), 0.0
    for r, (p, n) in enumerate(zip(prompts, n_new)):
        assert len(outs[r]) == len(p) + n and np.array_equal(outs[r][:len(p)], p)
        oracle.attend_over(stored[r])
        for i, t in enumerate(outs[r][:-1]):
            ref = logprobs(oracle.step(int(t)))
            worst = max(worst, float(np.abs(logprobs(rows[r][i]) - ref).max()))
            a, b = np.sort(ref)[-2:][::-1]
            if i + 1 >= len(p) and a - b > TIE:
                assert outs[r][i + 1] == int(ref.argmax()), (r, i)
    assert worst <= LOGPROB_TOL, worst


def test_a_request_is_the_same_in_any_company(model, small):
    m, s = model
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, small[0]["vocab"], n) for n in (8, 20, 4, 11)]
    together = m.generate(prompts, 10, s)
    for p, t in zip(prompts, together):
        assert np.array_equal(m.generate([p], 10, s)[0], t)


def test_running_out_of_pages_is_an_error(model, small):
    m, s = model
    with pytest.raises(RuntimeError, match="out of pages"):
        m.generate([[1] * 40] * 3, 8, s)  # three pages each, of eight
    with pytest.raises(ValueError):
        m.generate([[1] * 45], 8, s)
    assert len(m.generate([[1, 2]], 2, s)[0]) == 4  # usable after it


@pytest.mark.parametrize("rows, nh, nkv", [(1, 4, 1), (5, 16, 2), (33, 3, 3)])
def test_qk_rope_rows(fn, rows, nh, nkv):
    """fp32 sums of 256 squares and an angle reduced in double: 1e-6 of the row's largest value (its norm is 16)."""
    import torch
    rng = np.random.default_rng(rows)
    x = torch.from_numpy(rng.standard_normal((rows, nh * 512 + nkv * 256)).astype(np.float32)).cuda()
    wq, wk = (torch.from_numpy((1 + 0.1 * rng.standard_normal(256)).astype(np.float32)).cuda() for _ in range(2))
    inv = torch.from_numpy(np.asarray(rope_inv_freq(1e7), np.float32)).cuda()
    pos = rng.integers(0, 100_000, rows).astype(np.int32)
    pos[-1] = -1 if rows > 1 else 7
    q, k, ps = x[:, :nh * 512].view(rows, nh, 512), x[:, nh * 512:], x.shape[1]
    qo, ko = torch.full((rows, nh, 256), 9.0, device="cuda"), torch.full((rows, nkv, 256), 9.0, device="cuda")
    fn.qk_rope_rows(q.data_ptr(), ps, 512, k.data_ptr(), ps, 256, wq.data_ptr(), wk.data_ptr(), inv.data_ptr(),
                    torch.from_numpy(pos).cuda().data_ptr(), rows, nh, nkv, qo.data_ptr(), ko.data_ptr(), 1e-6,
                    torch.cuda.current_stream().cuda_stream)
    fn.sync(torch.cuda.current_stream().cuda_stream)
    f64 = lambda t: t.cpu().numpy().astype(np.float64)  # noqa: E731
    for got, src, w, n in ((qo, f64(q)[..., :256], f64(wq), nh), (ko, f64(k).reshape(rows, nkv, 256), f64(wk), nkv)):
        for i in range(rows):
            if pos[i] < 0:
                assert not got[i].any()
                continue
            want = rope(np.stack([rmsnorm(src[i, h], w, 1e-6) for h in range(n)]), int(pos[i]), f64(inv))
            assert np.abs(f64(got[i]) - want).max() <= 1e-6 * np.abs(want).max()


def test_gdn_reset_seq(fn):
    import torch
    rng = np.random.default_rng(2)
    nkh, nvh, B = 2, 4, 3
    ch = 2 * nkh * 128 + nvh * 128
    a = [(rng.standard_normal(s) * 0.5).astype(np.float32) for s in ((ch, 4), (nvh,), (nvh,), (128,))]
    h = fn.gdn_create_batch(nkh, nvh, a[0], a[1], -np.abs(a[2]), a[3], B)
    x = torch.from_numpy(rng.standard_normal((B, ch + nvh * 128 + 2 * nvh)).astype(np.float32)).cuda()
    out = torch.zeros(4, B, nvh * 128, device="cuda")
    s = torch.cuda.current_stream().cuda_stream

    def run(i):
        w = x.shape[1]
        fn.gdn_run_batch(h, x.data_ptr(), w, x.data_ptr() + 4 * ch, w, x.data_ptr() + 4 * (ch + nvh * 128), w, out[i].data_ptr(),
                         nvh * 128, 0, s)
    run(0)
    run(1)
    fn.gdn_reset_seq(h, 1, s)
    run(2)  # sequence 1 from zero again, the others a third token
    fn.sync(s)
    assert torch.equal(out[2, 1], out[0, 1]) and not torch.equal(out[2, 0], out[0, 0])
    fn.gdn_reset(h, s)
    run(3)
    fn.sync(s)
    assert torch.equal(out[3], out[0])
    for bad in (-1, B):
        with pytest.raises(RuntimeError, match="no such sequence"):
            fn.gdn_reset_seq(h, bad, s)
    fn.gdn_free(h)
