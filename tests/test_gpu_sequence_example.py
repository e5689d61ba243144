"""The example of the sequence operators trains and serves."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu


def test_mixer_learns_the_filter_and_serves(hip_ctx):
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import sequence_mixer
    losses, apart = sequence_mixer.main(60)
    # the filter's own energy is most of the first loss; a layer that mixes only within tokens cannot go below it
    assert losses[-1] < 0.5 * losses[0]
    # both ways round in 32 bits; torch's products of one token's rows and of all rows differ as much
    assert apart < 1e-5
