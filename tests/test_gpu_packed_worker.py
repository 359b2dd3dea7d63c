"""Workers whose training shard is held in 4 bits, with dropout, through the host parameter server:
the final theta against the same rounds on the CPU oracle, on the values the codes stand for and the
masks the seed gives."""
import json
import os
import subprocess

import numpy as np
import pytest

import mxfp_ref as ref

pytestmark = pytest.mark.gpu
PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "paracel_amd")


@pytest.fixture()
def server_info():
    p = subprocess.Popen([os.path.join(PKG, "plr_ps_server")], stdout=subprocess.PIPE, text=True)
    yield p.stdout.readline().strip()
    p.kill()
    p.wait()


def dropped(Q, worker, rd, rate, seed, first):
    from paracel_amd import Dropout

    k = ref.keep(Q.shape[0], Q.shape[1] - first, Dropout(rate, seed, rd, worker << 40))
    D = Q.copy()
    D[:, first:] *= k * ref.kept_scale(rate)
    return D


@pytest.mark.parametrize("workers", [1, 2])
def test_synthetic_rounds_with_dropout(server_info, oracle, gen, tmp_path, workers):
    n, d, rounds, rate, seed = 3000, 300, 12, 0.2, 77
    cfg = gen.configs()["c5_e2e_2m_x_512"].scaled(n)
    alpha, beta = 0.5 / n, 0.001
    out = tmp_path / "theta.bin"
    cmd = [os.path.join(PKG, "plr_lr_worker"), "--server_info", server_info, "--synthetic",
           "%x,%d,%d,%.17g" % (cfg.seed, n, d, cfg.spec.scale), "--rounds", str(rounds),
           "--alpha", "%.17g" % alpha, "--beta", "%.17g" % beta, "--theta0", "zero",
           "--update_file", os.path.join(PKG, "liblr_update.so"), "--theta_out", str(out),
           "--storage", "mxfp4", "--dropout", str(rate), "--dropout_seed", str(seed),
           "--worker_sz", str(workers)]
    ps = [subprocess.Popen(cmd + ["--worker_id", str(w)], stdout=subprocess.PIPE, stderr=subprocess.PIPE,
                           text=True) for w in range(workers)]
    for p in ps:
        o, e = p.communicate(timeout=110)
        assert p.returncode == 0, e
        assert "4-bit shard" in o
    spec = gen.GenSpec(cfg.seed, gen.NORMAL, 0, cfg.spec.scale, 0.0, 1.0)
    X = gen.gen_X(spec, 0, n, d)
    y = gen.gen_labels(spec, 0, X, gen.gen_vec(cfg.seed, gen.STREAM_THETA_STAR, d, gen.NORMAL, 1.0))
    Q, theta = ref.rounded(X), np.zeros(d)
    cut = [n * w // workers for w in range(workers + 1)]
    for rd in range(rounds):
        step = [oracle.dgd_delta(dropped(Q[a:b], w, rd, rate, seed, 0), y[a:b], theta, alpha, beta)
                for w, (a, b) in enumerate(zip(cut, cut[1:]))]
        theta = theta + sum(step)
    got = np.fromfile(out)
    assert np.linalg.norm(got - theta) <= 1e-10 * np.linalg.norm(theta)


@pytest.mark.parametrize("worker", ["plr_lr_worker", "plr_ridge_worker"])
def test_csv_workers(server_info, oracle, tmp_path, worker):
    # the cache the first run leaves behind holds the doubles, not the rounded values: a second
    # run without the key trains on them
    rng = np.random.default_rng(9)
    n, k = 300, 40
    F = np.round(rng.normal(size=(n, k)), 4)
    lab = (rng.random(n) < 0.5).astype(int)
    train = tmp_path / "train.csv"
    with open(train, "w") as f:
        for i in range(n):
            f.write(",".join("%.4f" % v for v in F[i]) + ",%d\n" % lab[i])
    X, y = np.hstack([np.ones((n, 1)), F]), lab.astype(float)
    Q = X.copy()
    Q[:, 1:] = ref.rounded(F)
    alpha, beta, rounds = 1e-3, 0.01, 8
    base = {"training_input": str(train), "test_input": str(train), "predict_input": str(train),
            "output": str(tmp_path) + "/", "update_file": os.path.join(PKG, "liblr_update.so"),
            "update_func": "lr_theta_update", "method": "dgd", "rounds": rounds, "alpha": alpha,
            "beta": beta, "debug": False}
    for extra in ({"storage": "mxfp4", "dropout": 0.3, "dropout_seed": 5}, {"storage": "mxfp4"}, {}):
        cfg, out = tmp_path / "cfg.json", tmp_path / "theta.bin"
        cfg.write_text(json.dumps({**base, **extra}))
        r = subprocess.run([os.path.join(PKG, worker), "--server_info", server_info, "--cfg_file", str(cfg),
                            "--theta0", "zero", "--theta_out", str(out)],
                           capture_output=True, text=True, timeout=110)
        assert r.returncode == 0, r.stderr
        assert ("4-bit shard" in r.stdout) == bool(extra)
        theta = np.zeros(k + 1)
        for rd in range(rounds):
            D = X if not extra else Q if "dropout" not in extra else dropped(Q, 0, rd, 0.3, 5, 1)
            if worker == "plr_lr_worker":
                theta = theta + oracle.dgd_delta(D, y, theta, alpha, beta)
            else:
                theta = theta + alpha * D.T @ (y - D @ theta) - 2 * alpha * beta * n * theta
        got = np.fromfile(out)
        assert np.linalg.norm(got - theta) <= 1e-10 * np.linalg.norm(theta)
