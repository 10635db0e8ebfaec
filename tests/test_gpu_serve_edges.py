"""Edges of the serving-step operators.  Tolerances are those of
``test_gpu_serve_ops`` (derived there)."""
import pytest

from test_gpu_serve_ops import BF, FP, attn_inputs, check_attn

pytestmark = pytest.mark.gpu


# A capped score is cap * tanh(score / cap), good to a few 2^-24 of the score, whatever the
# cap: below the f32 error of the score's own dot product, which the tolerance holds.
@pytest.mark.parametrize("softcap", [1e-3, 1.0, 1e3, 1e4, 1e5, 1e8, 3e38])
@pytest.mark.parametrize("lens,d,dtype", [([(1, 700), (3, 900)], 128, BF), ([(1, 700), (3, 900)], 64, FP),
                                          ([(130, 700), (1, 50)], 128, BF), ([(130, 700), (40, 300)], 64, FP),
                                          ([(130, 300)], 256, BF)])
def test_caps_far_from_the_scores(cuda, lens, d, dtype, softcap):
    check_attn(attn_inputs(cuda, lens, 8, 2, d, 16, dtype), max(n for n, _ in lens), softcap=softcap)
