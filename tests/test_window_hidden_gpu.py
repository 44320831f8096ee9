"""Windowed attention where a cache's places that no token sees any more hold large numbers."""
import numpy as np
import pytest

from test_window_attention_gpu import Step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["k", "v", "kv"])
@pytest.mark.parametrize("value", [1e12, -3e38, np.inf, np.nan])
@pytest.mark.parametrize("tokens,dim,window", [(1, 64, 150), (9, 96, 150), (40, 64, 150), (40, 80, 150), (300, 128, 150), (256, 40, 150),
                                               (40, 64, 5), (40, 96, 5), (32, 128, 1)])
def test_places_that_no_token_sees(hip, tokens, dim, window, value, which):
    """Between the sinks and the first token's window, and past a length, anything may lie."""
    def spoil(s):
        for b, n in enumerate(s.lengths):
            for a in (getattr(s, x) for x in which):
                a[b, s.sinks:n - tokens - window + 1] = value
                a[b, n:] = -value
    s = Step(hip, 2, tokens, 1010, 4, 2, dim, window, 5, [1010, 946], spoil=spoil)
    s.run()
    assert np.isfinite(s.check()).all()
