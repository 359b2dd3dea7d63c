"""Packed shards of so many rows that a workgroup goes through several tiles of several groups of
row sets, with the next one requested ahead, in every kind of pass."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


# Rows read once by the kernel for up to 8 blocks of 32 columns, up to 64, up to 256 (that one with
# dropout alone), and in two sweeps.  n is no multiple of anything: shares differ by one, and the last
# group ends behind the last row.
@pytest.mark.parametrize("n, d", [(1500001, 100), (150001, 1000), (40001, 4100), (12001, 8225)])
def test_many_groups(plr, n, d):
    from paracel_amd import Dropout

    piece = 2003
    times, rest = divmod(n, piece)
    rng = np.random.default_rng(d)
    P = rng.normal(size=(piece, d)) / np.sqrt(d)
    y, theta = (rng.random(piece) < 0.5) * 1.0, rng.normal(size=d) / 8

    def drop_at(i):
        return Dropout(0.5, 11, 4, (1 << 32) - 70000 + i * piece)

    # what the rows give one piece at a time, which is a tile or less to a workgroup
    plr.set_data(P, y)
    plr.pack_data()
    Q = plr.get_data()[0]
    linear = plr.predict_linear(theta)
    g, l, _ = plr.loss_grad(theta)
    want = [times * g, times * l]
    dropped = [0, 0]
    for i in range(times):
        plr.set_dropout(drop_at(i))
        g, l, _ = plr.loss_grad(theta)
        dropped = [dropped[0] + g, dropped[1] + l]
    plr.set_dropout(None)
    plr.set_data(P[:rest], y[:rest])
    plr.pack_data()
    g, l, _ = plr.loss_grad(theta)
    want = [want[0] + g, want[1] + l]
    plr.set_dropout(drop_at(times))
    g, l, _ = plr.loss_grad(theta)
    dropped = [dropped[0] + g, dropped[1] + l]
    plr.set_dropout(None)

    plr.alloc_data(n, d)
    for i in range(times + 1):
        m = piece if i < times else rest
        plr.set_data_chunk(i * piece, P[:m], y[:m])
    plr.pack_data()
    # A residual is at most 1, so a column's terms sum to at most the sum of its magnitudes (twice
    # that with dropout).  Either side is off by 2^-53 of it for every addition along one chain of
    # partial sums (rows of a thread, slots, workgroups: under 700), and by the residuals' own error,
    # a quarter of the dot product's: under 70 additions along one chain, of terms whose magnitudes
    # sum to 0.64 sqrt(d) / 8 < 8.  The loss is off by the dot products' whole error, against a mean
    # of 0.69.  2000 * 2^-52 covers both sides of either.
    most = (times + 1) * np.abs(Q).sum(0)

    def same(got, expect, factor):
        assert (np.abs(got[0] - expect[0]) <= 2000 * 2.0 ** -52 * factor * most).all()
        assert abs(got[1] - expect[1]) <= 2000 * 2.0 ** -52 * abs(expect[1])  # terms of one sign

    for _ in range(2):
        plr.set_dropout(None)
        same(plr.loss_grad(theta), want, 1)
        assert abs(plr.calc_loss(theta)[0] - want[1]) <= 2000 * 2.0 ** -52 * want[1]
        plr.set_dropout(drop_at(0))
        same(plr.loss_grad(theta), dropped, 2)
    z = plr.predict_linear(theta)
    for i in (0, 1, times // 2, times - 1):
        assert np.abs(z[i * piece:(i + 1) * piece] - linear).max() <= 2e-13
    assert np.abs(z[times * piece:] - linear[:rest]).max() <= 2e-13
