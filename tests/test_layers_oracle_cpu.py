"""The oracle of the operators around a recurrence, against differences: each gradient that it writes out is the derivative of the
value that it computes (float64, central differences along a random direction of each input)."""

import numpy as np
import pytest

from oracle import layers_oracle as O

H = 1e-6


def agree(loss, inputs, grads, rng, names):
    for n in names:
        v = rng.standard_normal(inputs[n].shape)
        up, down = ({**inputs, n: inputs[n] + s * H * v} for s in (1, -1))
        d = (loss(up) - loss(down)) / (2 * H)
        # third order terms H^2 and the roundings 2^-53 / H of the losses
        assert abs(d - (grads[n] * v).sum()) < 1e-7 * (1 + np.abs(grads[n]).sum()), n


@pytest.mark.parametrize("shape,par", [((5, 7), (7,)), ((2, 3, 4, 6), (4, 6))])
def test_layer_norm(shape, par):
    rng = np.random.default_rng(1)
    inp = dict(x=rng.standard_normal(shape) + 1, weight=rng.standard_normal(par), bias=rng.standard_normal(par))
    dy = rng.standard_normal(shape)
    r = O.layer_norm(**inp, dy=dy)
    agree(lambda i: (O.layer_norm(**i)["y"][0] * dy).sum(), inp, {k: r["d" + k][0] for k in inp}, rng, list(inp))


@pytest.mark.parametrize("S", [1, 2, 9])
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("silu", [False, True])
def test_short_conv(S, W, silu):
    rng = np.random.default_rng(S + W)
    inp = dict(x=rng.standard_normal((2, S, 5)), weight=rng.standard_normal((5, W)), bias=rng.standard_normal(5),
               x_initial=rng.standard_normal((2, W - 1, 5)))
    dy, dl = rng.standard_normal((2, S, 5)), rng.standard_normal((2, W - 1, 5))

    def loss(i):
        o = O.short_conv(**i, silu=silu)
        return (o["y"][0] * dy).sum() + (o["last"][0] * dl).sum()
    r = O.short_conv(**inp, silu=silu, dy=dy, dlast=dl)
    agree(loss, inp, {k: r["d" + k][0] for k in inp}, rng, list(inp))


@pytest.mark.parametrize("G", [None, 1, 2])
@pytest.mark.parametrize("softplus", [False, True])
def test_ssm_scan(G, softplus):
    rng = np.random.default_rng(3)
    B, S, D, N = 2, 6, 4, 3
    bc = (B, S, N) if G is None else (B, S, G, N)
    n = rng.standard_normal
    inp = dict(x=n((B, S, D)), dt=n((B, S, D)) if softplus else np.abs(n((B, S, D))), a=-np.exp(n((D, N))), b=n(bc), c=n(bc), skip=n(D),
               z=n((B, S, D)), dt_bias=n(D) if softplus else np.abs(n(D)), h_initial=n((B, D, N)))
    dy, dh = n((B, S, D)), n((B, D, N))

    def loss(i):
        o = O.ssm_scan(**i, softplus=softplus)
        return (o["y"][0] * dy).sum() + (o["h_last"][0] * dh).sum()
    r = O.ssm_scan(**inp, softplus=softplus, dy=dy, dh_last=dh)
    agree(loss, inp, {k: r["d" + k][0] for k in inp}, rng, list(inp))


def test_scan_goes_on_where_it_stopped():
    rng = np.random.default_rng(4)
    B, S, D, N = 1, 7, 3, 2
    n = rng.standard_normal
    x, dt, z, b, c, a = n((B, S, D)), n((B, S, D)), n((B, S, D)), n((B, S, N)), n((B, S, N)), -np.exp(n((D, N)))
    whole = O.ssm_scan(x, dt, a, b, c, z=z, softplus=True)
    cut = lambda s: dict(x=x[:, s], dt=dt[:, s], a=a, b=b[:, s], c=c[:, s], z=z[:, s], softplus=True)  # noqa: E731
    first = O.ssm_scan(**cut(slice(0, 3)))
    second = O.ssm_scan(**cut(slice(3, S)), h_initial=first["h_last"][0])
    assert np.allclose(np.concatenate([first["y"][0], second["y"][0]], 1), whole["y"][0], rtol=1e-13, atol=1e-13)
    assert np.allclose(second["h_last"][0], whole["h_last"][0], rtol=1e-13, atol=1e-13)
