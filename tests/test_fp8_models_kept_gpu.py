"""GPU: what the models with 8-bit dense weights and scores keep and give back."""

import gc

import numpy as np
import pytest
import torch

from synth import model_config, model_weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def small():
    cfg = model_config(small=True)
    return cfg, model_weights(cfg, 3)


def test_a_step_runs_on_the_stream_it_is_given(fn, small):
    """The default stream, whose handle is 0, among them; what launches on the current stream must meet the rest of the step there."""
    from model import BatchDecodeModel
    m = BatchDecodeModel(fn, *small, 2, max_ctx=8, dense="fp8")
    try:
        at = []
        m._launch_step = lambda s: at.append((s, torch.cuda.current_stream().cuda_stream))
        other = torch.cuda.Stream()
        for s in (0, other.cuda_stream):
            m.launch_step(s)
            with torch.cuda.stream(other):
                m.launch_step(s)
        assert at == [(0, 0)] * 2 + [(other.cuda_stream,) * 2] * 2
    finally:
        m.free()


@pytest.mark.parametrize("serve", [False, True])
@pytest.mark.parametrize("dense", ["gguf", "fp8"])
def test_free_gives_the_dense_weights_back(fn, small, dense, serve):
    from model import BatchDecodeModel
    from serve import ServeModel
    cfg, W = small

    def make():
        if serve:
            return ServeModel(fn, cfg, W, batch=2, pages=4, max_ctx=16, page_size=16, dense=dense)
        return BatchDecodeModel(fn, cfg, W, 2, max_ctx=16, dense=dense)

    def held():
        gc.collect()
        torch.cuda.synchronize()
        return torch.cuda.memory_allocated()

    make().free()  # (what a first model leaves: the planner's and the library's own)
    m = make()
    before = held()
    dense_bytes = sum(t.numel() for t in weights(m)) if dense == "fp8" else 0
    m.free()
    assert before - held() >= dense_bytes
    m.free()  # again is nothing


def weights(m):
    from fp8 import Fp8Weight
    found = [m.head, *(v for L in m.layers for v in L.values())]
    return [v.q for v in found if isinstance(v, Fp8Weight)]


@pytest.mark.parametrize("top", [0, 3])
def test_scores_of_what_was_finished_are_kept(fn, small, top):
    from serve import OutOfPages, ServeModel
    m, s = ServeModel(fn, *small, batch=3, pages=8, max_ctx=48, page_size=16), torch.cuda.Stream()
    m.capture(s)
    try:
        with pytest.raises(OutOfPages, match="out of pages") as e:
            m.generate([[1, 2], [1] * 40, [1] * 40, [1] * 40], [2, 8, 8, 8], s, scores=top)
        outs, scores = e.value.outs, e.value.scores
        alone, said = m.generate([[1, 2]], 2, s, scores=top)
        assert len(scores) == 4 and scores[3] is None and [o is None for o in outs] == [q is None for q in scores]
        assert np.array_equal(outs[0], alone[0])
        for got, want in zip(scores[0], said[0]):
            assert np.array_equal(got, want) and len(got) == 3
        with pytest.raises(OutOfPages) as e:
            m.generate([[1, 2], [1] * 40, [1] * 40, [1] * 40], [2, 8, 8, 8], s)
        assert e.value.scores is None
    finally:
        m.free()
