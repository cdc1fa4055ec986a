"""The cache in 8 bits with position encodings of a user's own: the append turns rows itself only where that is what the encoding's `rotate` does."""
import pytest
import torch

import cache8_refs as R
import replay_util as U
from conftest import seeded_tokens
from denno_beta_amd.parts.positions import NoPositions, RotaryHalves, RotaryPairs


@pytest.fixture(params=[pytest.param("host", id="host"), pytest.param("gpu", marks=pytest.mark.gpu, id="gpu")])
def device(request):
    if request.param == "host":
        with R.emulated():
            yield "cpu"
    else:
        yield "cuda:0"


class LongTable(RotaryPairs):
    """A table of more frequencies than are turned."""

    def bind(self, tensors, runtime):
        super().bind(tensors, runtime)
        self.freq = torch.cat([self.freq, torch.full((4,), 0.5, device=runtime.device)])

    def turn(self, src, dst, positions, n_vec, width, **layout):
        from denno_beta_amd.kernels import ops
        return ops.rotary(src, dst, positions, self.freq[:self.dims // 2].contiguous(), n_vec, self.dims, width, mag=self.mag, **layout)


class LeftAlone(RotaryHalves):
    """An encoding that has a table and turns nothing with it."""

    def rotate(self, q, k, ctx):
        return q, k


class WithoutAFactor:
    """An encoding that is no descendant of the framework's, with a table of its own and no factor on cos and sin."""
    rotates = graph_safe = True

    def __init__(self, inner):
        self.inner, self.dims, self.head_dim = inner, inner.dims, inner.head_dim

    @property
    def freq(self):
        return self.inner.freq

    def rotate(self, q, k, ctx):
        return self.inner.rotate(q, k, ctx)


def logits(device, position):
    """Of an engine of one turned layer (8 query heads over 2 key heads of 32, 16 entries turned) with this encoding in place of its own."""
    from test_cache8_engine import runner
    r = runner(device, "float32", use_graphs=False)
    inner = getattr(position, "inner", position)
    inner.bind({}, r.runtime)
    r.runtime.position = position
    return torch.cat(list(U.replay(r, U.chunk_trace([seeded_tokens(7, 20, 61), seeded_tokens(8, 5, 61)])).values()))


@pytest.mark.parametrize("own,same", [
    (lambda: LongTable(16, 50.0, 32), lambda: RotaryPairs(16, 50.0, 32)),
    (lambda: LeftAlone(32, 50.0, 32), NoPositions),
    (lambda: WithoutAFactor(RotaryPairs(32, 50.0, 32)), lambda: RotaryPairs(32, 50.0, 32)),
], ids=["a longer table", "a rotate of its own", "no factor"])
def test_encodings_of_a_users_own(device, own, same):
    """What one rounding more does (32-bit rows turned and then rounded to 8 bits, or from 64 bits at once) moves a logit by far less than a turn
    too many or too few."""
    got, want, other = logits(device, own()), logits(device, same()), logits(device, RotaryPairs(32, 7.0, 32))
    spread = want.std(dim=1, keepdim=True)
    assert ((got - want).abs() / spread).max() <= 0.1
    assert ((other - want).abs() / spread).max() > 0.3      # (that this layer's turn shows)
