"""The operators together: the decoder-layer example."""
import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
import latent_decoder_layer as ex  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("prompts,steps", [((70, 1, 200), 4), ((1,), 2), ((129, 64, 63, 5, 1, 33), 1)])
def test_layer(cuda_device, cache, prompts, steps):
    """The two forms round different intermediates to bf16 (kv and P v against q W and o W): a few 2^-9 of
    their operands each, 2^-5 of the largest value with room for the cancellation in sums of 512."""
    y, gap = ex.run(prompts, steps, cache, cuda_device)
    assert y.shape == (len(prompts), 512) and torch.isfinite(y).all() and y.abs().sum() > 0
    assert gap < 2 ** -5
