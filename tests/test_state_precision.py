"""What the bound on the delta rule's states tells apart, on a CPU model of its chunks: three parts of 8 bits a number keep it, any loss of
a part or of a product of parts does not."""
import numpy as np
import pytest

import attnref as R
import stateref as S

LOSSES = {"a part of the state": dict(parts=(2, 3, 3, 3)), "a part of V - K S": dict(parts=(3, 2, 3, 3)), "a part of the inverse": dict(parts=(3, 3, 2, 3)),
          "a part of the corrections": dict(parts=(3, 3, 3, 2)), "the product of the first and third": dict(skip=((0, 2),)),
          "of the second ones": dict(skip=((1, 1),)), "of the third and first": dict(skip=((2, 0),))}


def inputs(n, dk, kind, rng):
    k = rng.normal(size=(n, dk))
    k = R.rounded(k / np.sqrt((k * k).sum(-1, keepdims=True)), kind)
    v = R.rounded(rng.normal(size=(n, dk)) * S.STATE_VALUES, kind)
    g = (-np.abs(rng.normal(size=n)) * S.STATE_DECAY).astype(np.float32).astype(np.float64)
    return k, v, g, rng.uniform(0.2, 0.9, n).astype(np.float32), rng.normal(size=(dk, dk)).astype(np.float32)


@pytest.mark.parametrize("n", [64, 140, 300])
@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("kind", [R.M.BF16, R.M.F16])
def test_the_bound_on_states_needs_every_part(n, dk, kind):
    k, v, g, beta, state = inputs(n, dk, kind, np.random.default_rng(n + dk))
    _, _, want, _ = S.delta(k, k, v, g, beta, state, 1.0, 0.0, np.zeros(n), np.zeros(n))
    exact = kind == R.M.BF16
    assert S.state_norm_error(S.chunked(k, v, g, beta, state, exact), want) <= S.STATE_NORM
    for name, loss in LOSSES.items():
        assert S.state_norm_error(S.chunked(k, v, g, beta, state, exact, **loss), want) > 1.5 * S.STATE_NORM, name
