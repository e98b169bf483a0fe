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


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-9, 1e-14, 1e-16, 3e-18])
def test_small_gradients_beside_one_far_larger(size):
    """The same where all of them are small: 2^-22 of the neighbours is left by the pieces, and their dS is bounded by themselves."""
    f = case(1, 100, 1500, 1, 1, 64, None, seed=1)
    f["g"] *= np.float32(size)
    f["g"][0, 7] *= np.float32(2.0) ** 16
    _, dq, _ = evaluate(graph(False, None), f, ndarray.gpu(0))
    want = definition(f["q"], f["kv"], None, 0.125, f["g"])[0][1]
    assert (np.abs(dq - want).max(3) / np.abs(want).max(3)).max() <= 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-28, 1e-32, 1e-35])
@pytest.mark.parametrize("tq,d", [(100, 64), (100, 128), (1, 64)])
def test_gradients_of_next_to_nothing(size, tq, d):
    """Gradients near the end of fp32 do not vanish: their pieces and dS keep 2^-19 of the largest number of a row at the least,
    and some hundred of such errors add up."""
    f = case(2, tq, 130, 2, 1, d, None, seed=2)
    f["g"] = f["g"] * np.float32(size)
    _, dq, dkv = evaluate(graph(False, None), f, ndarray.gpu(0))
    want = definition(f["q"], f["kv"], None, d ** -0.5, f["g"])[0]
    for got, w in ((dq, want[1]), (dkv[:, :, 0], want[2][:, :, 0]), (dkv[:, :, 1], want[2][:, :, 1])):
        # (what is below 2^-126, of g or of a result, counts as 0 in every kernel)
        assert np.abs(got - w).max() <= 1e-4 * np.abs(w).max() + 4 * 2.0 ** -126


@pytest.mark.gpu
@pytest.mark.parametrize("tq,d", [(1, 64), (40, 64), (140, 128)])
@pytest.mark.parametrize("size", [1e33, 1e36])
def test_values_near_the_largest_number(tq, d, size):
    """A result is a mean of values, so it is a number where they are; so are the gradients of small enough ones."""
    f = case(2, tq, 150, 2, 1, d, "holes", seed=4)
    f["kv"][:, :, 1] *= np.float32(size) / np.abs(f["kv"][:, :, 1]).max()
    f["g"] = f["g"] * np.float32(1e-37)
    got = evaluate(graph(True, None), f, ndarray.gpu(0))
    g = np.where(np.abs(f["g"]) < 2.0 ** -126, 0, f["g"])             # (which count as 0 in every kernel)
    for a, b, t in zip(got, *definition(f["q"], f["kv"], f["key"], d ** -0.5, g)):
        assert np.isfinite(a).all() and np.all(np.abs(a - b) <= t + 4 * 2.0 ** -126)
