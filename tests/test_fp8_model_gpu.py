"""GPU: the batched decode step with 8-bit dense weights (BatchDecodeModel, ServeModel dense="fp8") and the scores that
ServeModel.generate returns.

Tolerances. Scores against the oracle on the very logits that the step left: those of tests/test_logprobs_gpu.py. The 8-bit step against the
step in the file's formats: a rounding to e4m3 is off by up to 2^-4 of a value, evenly spread, so 2^-4 / sqrt(3) = 3.6% in the root mean
square at the most, for rows as for weights: 5.1% of a projection's output if errors of its terms do not cancel, less where they do as terms
do. The small model has four layers of two such projections and the head: 5.1% sqrt(9) = 15% of the logits if every one's errors
reached them whole and norms kept their proportion; twice that is allowed for what gates and experts (a router's choice may turn)
make of them, 30%, as a root mean square over all rows, which is what was reckoned (a single row whose router turned is off by more). A
projection left out, or of another layer, is off by 100% and more. What each part of the step computes is tested apart, from the values
that it was given, with the tolerances of tests/test_fp8_gpu.py.
"""

import numpy as np
import pytest

from oracle import logprobs as O
from synth import model_config, model_weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def small():
    cfg = model_config(small=True)
    return cfg, model_weights(cfg, 3)


def steps(fn, model, prompts, n):
    """The logits of n steps of a batched model, eager, from its prompts [B][>= n]."""
    import torch
    s = torch.cuda.Stream()
    model.start(prompts, s)
    got = []
    for _ in range(n):
        model.launch_step(s.cuda_stream)
        fn.sync(s.cuda_stream)
        got.append(model.logits.double().cpu().numpy())
    return np.stack(got)


@pytest.mark.parametrize("batch", [1, 5])
def test_dense_fp8_step(fn, small, batch):
    import torch
    from model import BatchDecodeModel
    cfg, W = small
    rng = np.random.default_rng(batch)
    prompts = rng.integers(0, cfg["vocab"], (batch, 6))
    a = BatchDecodeModel(fn, cfg, W, batch, max_ctx=16)
    b = BatchDecodeModel(fn, cfg, W, batch, max_ctx=16, dense="fp8")
    try:
        x, y = steps(fn, a, prompts, 6), steps(fn, b, prompts, 6)
        x, y = x - x.mean(-1, keepdims=True), y - y.mean(-1, keepdims=True)
        assert 1e-3 < np.linalg.norm(y - x) / np.linalg.norm(x) <= 0.30
        # the graph gives the eager step's bits, and every place the same
        s = torch.cuda.Stream()
        same = np.repeat(prompts[:1], batch, 0)
        eager = steps(fn, b, same, 6)
        assert (eager == eager[:, :1]).all()
        b.capture(s)
        b.start(same, s)
        for i in range(6):
            with torch.cuda.stream(s):
                b.graph.replay()
            fn.sync(s.cuda_stream)
            assert np.array_equal(b.logits.double().cpu().numpy(), eager[i])
    finally:
        a.free()
        b.free()


def test_dense_fp8_parts(fn, small):
    """Every layer's projections and norms, and the head, from given rows: the weights are the file's values in 8 bits."""
    import torch
    from model import BatchDecodeModel
    from oracle import dequant as D
    from oracle import fp8 as F
    cfg, W = small
    B, d, P = 3, cfg["D"], cfg["proj"]
    np64 = lambda t: t.double().cpu().numpy()  # noqa: E731
    m = BatchDecodeModel(fn, cfg, W, B, max_ctx=8, dense="fp8")

    def weight(qtype, raw):
        _, qk, block = D.TYPES[qtype]
        return F.groups(D.dequant_rows(raw, qtype, len(raw), raw.shape[1] // block * qk), 128)

    def close(got, rows, qw):
        want, size = F.product(*rows, *qw)
        assert (np.abs(got - want) <= 2.0 ** -14 * size).all()

    try:
        s = torch.cuda.current_stream().cuda_stream
        g = torch.Generator(device="cuda")
        g.manual_seed(7)
        fill = lambda t: t.copy_(torch.randn(t.shape, device="cuda", generator=g))  # noqa: E731
        for L, w in zip(m.layers, W["layers"]):
            fill(m.h)
            h, norm = np64(m.h), np64(L["norm1"])
            m._norm(L["norm1"], s)
            rows = F.groups(F.rms(h, norm, cfg["eps"]), 1)
            assert np.array_equal(np64(m.rows8[d].q), rows[0]) and np.array_equal(np64(m.rows8[d].scale), rows[1])
            kind = L["kind"] == "G"
            raw = np.concatenate([w[n] for n in (("w_in", "w_ab") if kind else ("w_q", "w_k", "w_v"))])
            m.proj.fill_(5)
            m._project(L["w_in"] if kind else L["w_qkv"], m.proj, s)
            fn.sync(s)
            close(np64(m.proj)[:, :len(raw)], rows, weight(P, raw))
            assert (np64(m.proj)[:, len(raw):] == 5).all()
            mix, out = (m.core, "w_out") if kind else (m.att, "w_o")
            fill(mix)
            m._join(L["w_out"] if kind else L["w_o"], mix, L["norm2"], s)
            fn.sync(s)
            close(np64(m.y), F.groups(np64(mix), 1), weight(P, w[out]))
            total = (h.astype(np.float32) + np64(m.y).astype(np.float32)).astype(np.float64)
            assert np.array_equal(np64(m.h), total)
            assert np.array_equal(np64(m.x), F.rms(total, np64(L["norm2"]), cfg["eps"]).astype(np.float64))
        m._norm(m.final_norm, s)
        m._project(m.head, m.logits, s)
        fn.sync(s)
        close(np64(m.logits), F.groups(F.rms(total, np64(m.final_norm), cfg["eps"]), 1), weight(cfg["head"], W["head"]))
    finally:
        m.free()


def test_dense_refuses(fn, small):
    from model import BatchDecodeModel
    with pytest.raises(ValueError, match="dense"):
        BatchDecodeModel(fn, *small, 2, dense="int8")


@pytest.mark.parametrize("dense", ["gguf", "fp8"])
@pytest.mark.parametrize("top", [0, 4])
def test_serve_scores(fn, small, dense, top):
    import torch
    from serve import ServeModel
    cfg, W = small
    m = ServeModel(fn, cfg, W, batch=3, pages=12, max_ctx=48, page_size=16, dense=dense)
    try:
        s = torch.cuda.Stream()
        m.capture(s)
        rng = np.random.default_rng(top)
        prompts = [rng.integers(0, cfg["vocab"], n) for n in (5, 1, 9, 3)]
        n_new = [3, 7, 1, 4]
        rows = {}
        keep = lambda r, i, row: rows.__setitem__((r, i), row.double().cpu().numpy())  # noqa: E731
        outs, scores = m.generate(prompts, n_new, s, logits=keep, scores=top)
        plain = m.generate(prompts, n_new, s)
        for r, (p, n) in enumerate(zip(prompts, n_new)):
            assert np.array_equal(outs[r], plain[r]) and len(outs[r]) == len(p) + n
            q = scores[r]
            assert q.logprob.shape == q.rank.shape == q.entropy.shape == (len(outs[r]) - 1,)
            assert q.top_ids.shape == q.top_logprobs.shape == (len(outs[r]) - 1, top)
            for i in range(len(outs[r]) - 1):
                logprob, rank, entropy, ids, logs = O.row(rows[r, i], int(outs[r][i + 1]), top)
                big = np.abs(rows[r, i]).max()
                assert abs(q.logprob[i] - logprob) <= 2.0 ** -20 + 2.0 ** -22 * big and q.rank[i] == rank
                assert abs(q.entropy[i] - entropy) <= 2.0 ** -19 + 2.0 ** -20 * entropy
                assert np.array_equal(q.top_ids[i], ids) and (np.abs(q.top_logprobs[i] - logs) <= 2.0 ** -20 + 2.0 ** -22 * big).all()
                if i + 1 >= len(p):  # greedy: the token is the first of its row
                    assert q.rank[i] == 0 and (top == 0 or q.top_ids[i][0] == outs[r][i + 1])
        with pytest.raises(ValueError, match="scores"):
            m.generate(prompts, n_new, s, scores=33)
    finally:
        m.free()


def test_a_prompt_scored_in_8_bits(fn):
    """Residual, norm, 8-bit head and scores of a prompt's rows, as a scoring pass strings them together, against the oracles."""
    import fp8
    import logprobs
    import torch
    from oracle import fp8 as F
    rows, d, vocab = 300, 512, 5003
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    h, y, norm, w = rand(rows, d).bfloat16(), rand(rows, d).bfloat16(), 1 + 0.1 * rand(d), rand(vocab, d) * 0.1
    tok = torch.randint(vocab, (rows,), device="cuda", generator=g).int()
    head = fp8.Fp8Weight.quantise(fn, w)
    total = (h.float() + y.float()).bfloat16().double().cpu().numpy()
    x = fp8.quantise_rows(fn, h, add=y, total=h, weight=norm)
    logits = head.product(x)
    got = logprobs.token_logprobs(fn, logits, tok, top=3)
    fn.sync(torch.cuda.current_stream().cuda_stream)
    assert np.array_equal(h.double().cpu().numpy(), total)
    q, s = F.groups(F.rms(total, norm.double().cpu().numpy(), 1e-6), 1)
    assert np.array_equal(x.q.double().cpu().numpy(), q) and np.array_equal(x.scale.double().cpu().numpy(), s)
    wq, ws = F.groups(w.double().cpu().numpy(), 128)
    want, size = F.product(q, s, wq, ws)
    z = logits.double().cpu().numpy()
    assert (np.abs(z - want) <= 2.0 ** -14 * size).all()  # tests/test_fp8_gpu.py
    said = O.rows(z, tok.tolist(), 3)
    assert np.array_equal(got.rank.cpu().numpy(), said["rank"]) and np.array_equal(got.top_ids.cpu().numpy(), said["top_ids"])
    assert np.abs(got.logprob.double().cpu().numpy() - said["logprob"]).max() <= 2.0 ** -20 + 2.0 ** -22 * np.abs(z).max()
