"""GPU: what the models with 8-bit dense weights and scores keep and give back."""

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
