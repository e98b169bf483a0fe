"""How exact the attention across is where rows of one tile of 128 differ by more than an fp16 pair spans: the bounds that the
operator states, against the definition in 64 bits."""
import numpy as np
import pytest

from tsplit_b200 import ndarray
from test_cross_attention import case, check, definition, evaluate, graph


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["q", "k", "v", "g"])
@pytest.mark.parametrize("power", [16, 20, 24, 30])
@pytest.mark.parametrize("tq,tk,d", [(150, 260, 64), (140, 130, 128), (1, 260, 64)])
def test_one_row_far_larger_than_its_neighbours(which, power, tq, tk, d):
    """Element by element within 2^-22 of a number or 2^-38 of the largest one of its tile, carried through the formulas."""
    f = case(2, tq, tk, 2, 1, d, "holes", seed=power)
    f["key"][:, 3] = 1
    at = (f["q"] if which == "q" else f["g"])[:, tq // 2] if which in "qg" else f["kv"][:, 3, "kv".index(which)]
    at *= np.float32(2.0) ** power
    # scores stay within some hundreds, as they do wherever a soft-max is of use
    check(f, ndarray.gpu(0), scale=d ** -0.5 * (2.0 ** -power if which in "qk" else 1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("power,most", [(12, 4e-6), (20, 6e-5), (24, 1e-3)])
@pytest.mark.parametrize("tk,d", [(130, 64), (1500, 64), (1500, 128)])
def test_gradients_of_queries_beside_one_far_larger(power, most, tk, d):
    """The rows beside it keep what 2^-38 of the larger row leaves of them: 2^(power - 38) relative to their own numbers, times
    some ten for the sums over 64 columns and 130 keys (16 steps of 2^-22 at the least); no less where there are more keys."""
    f = case(1, 100, tk, 1, 1, d, None, seed=1)
    f["g"][0, 7] *= np.float32(2.0) ** power
    _, dq, _ = evaluate(graph(False, None), f, ndarray.gpu(0))
    want = definition(f["q"], f["kv"], None, d ** -0.5, f["g"])[0][1]
    off = np.abs(dq - want).max(3) / np.abs(want).max(3)
    assert off[0, 7, 0] <= 4e-6 and np.delete(off[0, :, 0], 7).max() <= most
