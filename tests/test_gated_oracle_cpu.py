"""The oracle of the gated linear recurrence against differences, and its generator against published words."""

import numpy as np
import pytest

from oracle import gated_oracle as O
from test_layers_oracle_cpu import agree


@pytest.mark.parametrize("scale", [None, "convex", "variance"])
@pytest.mark.parametrize("rate", [False, True])
@pytest.mark.parametrize("i,z", [(False, False), (True, False), (False, True), (True, True)])
def test_gradients(scale, rate, i, z):
    rng = np.random.default_rng(3)
    n = rng.standard_normal
    B, S, D = 2, 6, 4
    inp = dict(x=n((B, S, D)), f=n((B, S, D)), h_initial=n((B, D)))
    if i:
        inp["i"] = n((B, S, D))
    if z:
        inp["z"] = n((B, S, D))
    if rate:
        inp["rate"] = -np.exp(n(D))
    dy, dh = n((B, S, D)), n((B, D))

    def loss(k):
        o = O.gated_scan(**k, input_scale=scale)
        return (o["y"][0] * dy).sum() + (o["h_last"][0] * dh).sum()
    r = O.gated_scan(**inp, input_scale=scale, dy=dy, dh_last=dh)
    agree(loss, inp, {k: r["d" + k][0] for k in inp}, rng, list(inp))


@pytest.mark.parametrize("rate", [None, np.array([-0.01, -2.0])])
def test_goes_on_where_it_stopped_and_starts_anew(rate):
    rng = np.random.default_rng(4)
    x, f = rng.standard_normal((1, 9, 2)), rng.standard_normal((1, 9, 2))
    whole = O.gated_scan(x, f, rate=rate, input_scale="convex")
    first = O.gated_scan(x[:, :4], f[:, :4], rate=rate, input_scale="convex")
    second = O.gated_scan(x[:, 4:], f[:, 4:], rate=rate, h_initial=first["h_last"][0], input_scale="convex")
    assert np.allclose(np.concatenate([first["y"][0], second["y"][0]], 1), whole["y"][0], rtol=1e-13, atol=1e-13)
    if rate is None:
        f[:, 4] = -700.0
        assert np.allclose(O.gated_scan(x, f)["y"][0][:, 4:], O.gated_scan(x[:, 4:], f[:, 4:])["y"][0], rtol=1e-13, atol=1e-13)


# words of the generator as its authors' test vectors have them (kat_vectors of Random123)
VECTORS = [(7, "00000000 00000000 00000000 00000000", "00000000 00000000", "5f6fb709 0d893f64 4f121f81 4f730a48"),
           (7, "ffffffff ffffffff ffffffff ffffffff", "ffffffff ffffffff", "5207ddc2 45165e59 4d8ee751 8c52f662"),
           (10, "00000000 00000000 00000000 00000000", "00000000 00000000", "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
           (10, "ffffffff ffffffff ffffffff ffffffff", "ffffffff ffffffff", "408f276d 41c83b0e a20bc7c6 6d5451fd")]


@pytest.mark.parametrize("rounds,counter,key,words", VECTORS)
def test_generator(rounds, counter, key, words):
    split = lambda s: np.array([int(w, 16) for w in s.split()], dtype=np.uint64)  # noqa: E731
    assert np.array_equal(O.philox4x32(split(counter), split(key), rounds), split(words))


def test_kept_elements_are_those_of_the_whole():
    whole = O.kept((40, 33), 0.3, 12345, 7)
    assert np.array_equal(O.kept((100,), 0.3, 12345, 7, first=501), whole.reshape(-1)[501:601])
    # 1320 draws: six deviations of a share of 0.7
    assert abs(whole.mean() - 0.7) < 6 * (0.21 / whole.size) ** 0.5
    assert O.kept((1000,), 0.0, 1).all() and not O.kept((1000,), 1.0, 1).any()
