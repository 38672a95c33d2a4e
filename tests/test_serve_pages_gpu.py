"""GPU: ServeModel with fewer pages than its requests may want: they wait for pages, or what was finished is kept."""

import numpy as np
import pytest

from synth import model_config, model_weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def small():
    cfg = model_config(small=True)
    return cfg, model_weights(cfg, 3)


def serve(fn, small, pages):
    import torch
    from serve import ServeModel
    m, s = ServeModel(fn, *small, batch=3, pages=pages, max_ctx=48, page_size=16), torch.cuda.Stream()
    m.capture(s)
    return m, s


@pytest.fixture(scope="module")
def model(fn, small):
    m, s = serve(fn, small, 8)
    yield m, s
    m.free()


def test_requests_wait_for_pages(model, small):
    """Three pages each, of eight: two at a time; then lengths of all kinds. Each is the same as alone."""
    m, s = model
    rng = np.random.default_rng(0)
    for lengths, n_new in (([40, 40, 40], 8), ([40, 3, 17, 33, 1, 40, 16], [8, 30, 16, 2, 1, 8, 20])):
        prompts = [rng.integers(0, small[0]["vocab"], n) for n in lengths]
        together = m.generate(prompts, n_new, s, wait=True)
        n_new = [n_new] * len(prompts) if np.ndim(n_new) == 0 else n_new
        for p, n, t in zip(prompts, n_new, together):
            assert len(t) == len(p) + n and np.array_equal(m.generate([p], n, s)[0], t)


def test_what_was_finished_is_kept(model):
    from serve import OutOfPages
    m, s = model
    with pytest.raises(OutOfPages, match="out of pages") as e:
        m.generate([[1, 2], [1] * 40, [1] * 40, [1] * 40], [2, 8, 8, 8], s)
    assert np.array_equal(e.value.outs[0], m.generate([[1, 2]], 2, s)[0])
    assert len(e.value.outs) == 4 and e.value.outs[3] is None


def test_a_request_that_never_fits_is_refused_at_once(fn, small):
    m, s = serve(fn, small, 4)
    with pytest.raises(ValueError, match="more pages"):
        m.generate([[1], [1] * 40], 8, s, wait=True)
    assert len(m.generate([[1] * 20], 8, s, wait=True)[0]) == 28
    m.free()
