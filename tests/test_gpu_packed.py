"""The passes over a shard held in 4 bits, with and without dropout, against the CPU oracle on the
values the codes stand for (the bar of the double-precision passes, 1e-10, holds here too: the
arithmetic is in 64 bits), and the gradient against differences of the loss."""
import numpy as np
import pytest

import mxfp_ref as ref

pytestmark = pytest.mark.gpu

REL = 1e-11

SHAPES = [(1, 1), (5, 2), (1000, 31), (777, 32), (64, 33), (5000, 41), (3000, 100), (1234, 257),
          (2500, 512), (1001, 1000), (999, 1100), (300, 2049), (257, 2080), (130, 4100), (67, 8193),
          (40, 16384), (90, 2080), (60, 4097), (70, 8160), (50, 8193), (33, 16385), (21, 20000), (3, 40001), (1, 1000), (20000, 3), (700, 15361), (200, 30000)]


def close(got, want, rel=REL):
    got, want = np.asarray(got), np.asarray(want)
    assert np.linalg.norm(got - want) <= rel * max(np.linalg.norm(want), 1e-300), (
        np.linalg.norm(got - want), np.linalg.norm(want))


def shard(n, d, seed=0):
    rng = np.random.default_rng(n * 1009 + d + seed)
    X = rng.normal(size=(n, d)) / np.sqrt(d) * 2.0 ** rng.integers(-2, 3, size=(n, 1))
    X[rng.random((n, d)) < 0.2] = 0.0
    y = (rng.random(n) < 0.5) * 1.0
    theta = rng.normal(size=d)
    return X, y, theta


def expect(oracle, X, y, theta, flags):
    """(gradient sum, loss sum) by the oracle, or plainly for the formulas it does not have."""
    z = X @ theta
    if flags == 3:
        return X.T @ (z - y), float(((z - y) ** 2).sum())
    g = oracle.gsum(X, y, theta)
    if flags == 0:
        return g, oracle.calc_loss_sum(X, y, theta)
    s = np.where(y == 1, -z, z)
    return g, float((np.log1p(np.exp(-np.abs(s))) + np.maximum(s, 0)).sum()) if flags == 1 else 0.0


@pytest.mark.parametrize("n, d", SHAPES)
def test_passes(plr, oracle, n, d):
    X, y, theta = shard(n, d)
    plr.set_data(X, y)
    plr.pack_data()
    assert "4-bit" in plr.kernel_info() and plr.shape == (n, d)
    Q = ref.rounded(X)
    got_X, got_y = plr.get_data()
    assert np.array_equal(got_X, Q) and np.array_equal(got_y, y)
    for flags in (0, 1, 2, 3):
        g, loss, rows = plr.loss_grad(theta, flags)
        want, wl = expect(oracle, Q, y, theta, flags)
        close(g, want)
        close(loss, wl)
        assert rows == n
        if flags != 2:
            close(plr.calc_loss(theta, flags)[0], wl)
    delta, _ = plr.dgd_delta(theta, 0.01, 0.1)
    close(delta, oracle.dgd_delta(Q, y, theta, 0.01, 0.1))
    z = Q @ theta
    close(plr.predict_linear(theta), z)
    close(plr.predict(theta), 1 / (1 + np.exp(-z)))
    # bit for bit the same again
    assert np.array_equal(plr.loss_grad(theta)[0], plr.loss_grad(theta)[0])


@pytest.mark.parametrize("n, d", SHAPES)
@pytest.mark.parametrize("rate", [0.1, 0.5])
def test_dropout(plr, oracle, n, d, rate):
    from paracel_amd import Dropout

    X, y, theta = shard(n, d)
    plr.set_data(X, y)
    plr.pack_data()
    drop = Dropout(rate, 0xABCDEF0123456789, 12, (1 << 32) - 100)
    plr.set_dropout(drop)
    D = ref.rounded(X) * ref.keep(n, d, drop) * ref.kept_scale(rate)
    for flags in (0, 3):
        g, loss, _ = plr.loss_grad(theta, flags)
        want, wl = expect(oracle, D, y, theta, flags)
        close(g, want)
        close(loss, wl)
    # what does not make a gradient never drops
    close(plr.predict_linear(theta), ref.rounded(X) @ theta)
    plr.set_dropout(None)
    close(plr.loss_grad(theta)[0], expect(oracle, ref.rounded(X), y, theta, 0)[0])


@pytest.mark.parametrize("n, d", [(500, 2), (300, 42), (400, 101), (300, 257), (50, 2049), (30, 16386)])
def test_constant_first_column(plr, oracle, n, d):
    from paracel_amd import Dropout

    X, y, theta = shard(n, d, 5)
    X[:, 0] = 1.0
    plr.set_option("first_column_is_one", 1)
    plr.set_data(X, y)
    plr.pack_data()
    Q = X.copy()
    Q[:, 1:] = ref.rounded(X[:, 1:])
    assert np.array_equal(plr.get_data()[0], Q)
    g, loss, _ = plr.loss_grad(theta)
    close(g, oracle.gsum(Q, y, theta))
    close(loss, oracle.calc_loss_sum(Q, y, theta))
    drop = Dropout(0.3, 1, 2, 3)
    plr.set_dropout(drop)
    D = Q.copy()
    D[:, 1:] *= ref.keep(n, d - 1, drop) * ref.kept_scale(0.3)
    g, loss, _ = plr.loss_grad(theta)
    close(g, oracle.gsum(D, y, theta))
    close(loss, oracle.calc_loss_sum(D, y, theta))


@pytest.mark.parametrize("n, d", [(700, 100), (300, 1000), (20, 16400)])
def test_training_rounds(plr, oracle, n, d):
    from paracel_amd import Dropout

    X, y, theta = shard(n, d, 1)
    plr.set_data(X, y)
    plr.pack_data()
    Q = ref.rounded(X)
    drop = Dropout(0.25, 77, 40)
    for dr in (None, drop):
        plr.set_dropout(dr)
        th, curve = plr.train_dgd(theta, 0.05, 0.01, 6, want_curve=True)
        want, losses = theta.copy(), []
        for rd in range(6):
            D = Q if dr is None else Q * ref.keep(n, d, Dropout(0.25, 77, 40 + rd)) * ref.kept_scale(0.25)
            losses.append(oracle.calc_loss_sum(D, y, want))
            want = want + oracle.dgd_delta(D, y, want, 0.05, 0.01)
        close(th, want)
        close(curve, losses)


def test_gradient_against_differences(plr):
    from paracel_amd import Dropout

    X, y, theta = shard(400, 130, 2)
    plr.set_data(X, y)
    plr.pack_data()
    for drop in (None, Dropout(0.4, 9, 1)):
        plr.set_dropout(drop)
        g = plr.loss_grad(theta, 1)[0]
        for j in (0, 31, 32, 100, 129):
            h = 1e-5
            e = np.zeros_like(theta)
            e[j] = h
            up, down = plr.loss_grad(theta + e, 1)[1], plr.loss_grad(theta - e, 1)[1]
            # central difference: h^2 / 6 of a third derivative (at most sum |x|^3 / 10 ~ 10), and
            # 2^-52 of a loss of a few hundred over h
            assert abs((up - down) / (2 * h) - g[j]) < 1e-7


def test_empty_shard_and_refusals(plr):
    from paracel_amd import Dropout, PlrError

    with pytest.raises(PlrError) as e:
        plr.pack_data()
    assert e.value.code == -4
    plr.set_data(np.zeros((0, 40)), np.zeros(0))
    plr.pack_data()
    g, loss, n = plr.loss_grad(np.ones(40))
    assert n == 0 and loss == 0 and not g.any()
    X, y, theta = shard(50, 40)
    plr.set_data(X, y)  # a shard of doubles again
    plr.set_dropout(Dropout(0.5, 1))
    for call in (lambda: plr.loss_grad(theta), lambda: plr.dgd_delta(theta, 0.1, 0.1),
                 lambda: plr.train_dgd(theta, 0.1, 0.1, 2)):
        with pytest.raises(PlrError) as e:
            call()
        assert e.value.code == -5 and "pack" in str(e.value)
    plr.calc_loss(theta)
    plr.set_dropout(Dropout(0.0, 1))  # drops nothing: none
    plr.loss_grad(theta)
    plr.set_dropout(Dropout(0.5, 1))
    plr.pack_data()
    plr.pack_data()  # packed already: nothing to do
    plr.loss_grad(theta)
    with pytest.raises(PlrError) as e:
        plr.set_data_chunk(0, X, y)
    assert e.value.code == -5 and "4 bits" in str(e.value)
    for bad in (Dropout(1.0, 1), Dropout(-0.1, 1), Dropout(float("nan"), 1), Dropout(0.5, 1, 0, -1)):
        with pytest.raises(PlrError) as e:
            plr.set_dropout(bad)
        assert e.value.code == -1


def test_values_that_are_not_finite(plr):
    X, y, theta = shard(200, 70)
    X[11, 5] = np.nan
    X[60, 69] = np.inf
    plr.set_data(X, y)
    plr.pack_data()
    z = plr.predict_linear(theta)
    assert np.isnan(z[[11, 60]]).all() and np.isfinite(np.delete(z, [11, 60])).all()
    assert np.isnan(plr.loss_grad(theta)[1])


@pytest.mark.parametrize("n, d", [(300, 38), (250, 70), (200, 1000), (150, 4100), (40, 16400), (30, 20001)])
def test_a_nan_that_is_dropped_whole(plr, oracle, n, d):
    # a block with a NaN stands for NaN, but where nothing of it is kept it counts 0 like any other
    from paracel_amd import Dropout

    X, y, theta = shard(n, d, 3)
    drop = Dropout(0.97, 31, 1, 5)
    keep = ref.keep(n, d, drop)
    hit = 0
    for i in range(n):
        gone = [b for b in range(0, d, 32) if not keep[i, b:b + 32].any()]
        if gone:
            X[i, gone[i % len(gone)] if i % 3 else gone[-1]] = (np.nan, np.inf)[i % 2]
            hit += 1
    assert hit > n // 4
    plr.set_data(X, y)
    plr.pack_data()
    plr.set_dropout(drop)
    D = np.where(keep, ref.rounded(X), 0) * ref.kept_scale(0.97)
    g, loss, _ = plr.loss_grad(theta, 3)
    want, wl = expect(oracle, D, y, theta, 3)
    close(g, want)
    close(loss, wl)
    # one that is kept makes the loss NaN
    i, j = np.argwhere(keep)[len(np.argwhere(keep)) // 2]
    X[i, j] = np.nan
    plr.set_data(X, y)
    plr.pack_data()
    assert np.isnan(plr.loss_grad(theta, 3)[1])


def test_rows_of_every_layout_pack_alike(plr):
    # row-tiled, half-wave and streaming shards of doubles hold their rows differently
    for d in (7, 63, 64, 65, 96, 97, 130):
        X, y, _ = shard(333, d)
        plr.set_data(X, y)
        plr.pack_data()
        assert np.array_equal(plr.get_data(10, 200)[0], ref.rounded(X)[10:210])
