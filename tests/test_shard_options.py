"""The worker drivers' optional keys for 4-bit storage and dropout: what they refuse, before anything
is loaded or the GPU is touched (so this runs without one)."""
import json
import os
import subprocess

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "paracel_amd")
CFG = {"training_input": "none", "test_input": "", "predict_input": "", "output": "none/",
       "update_file": "none", "update_func": "lr_theta_update", "method": "dgd", "rounds": 1,
       "alpha": 0.1, "beta": 0.1, "debug": False}

BAD = [({"storage": "fp4"}, "storage must be"), ({"dropout": 0.5}, "needs storage mxfp4"),
       ({"storage": "f64", "dropout": 0.5}, "needs storage mxfp4"),
       ({"storage": "mxfp4", "dropout": 1.0}, "dropout must be"),
       ({"storage": "mxfp4", "dropout": -0.1}, "dropout must be"),
       ({"storage": "mxfp4", "dropout": "half"}, "dropout must be"),
       ({"storage": "mxfp4", "dropout_seed": "x"}, "dropout_seed must be")]


@pytest.mark.parametrize("worker", ["plr_lr_worker", "plr_ridge_worker"])
@pytest.mark.parametrize("extra, what", BAD)
def test_refusals(tmp_path, worker, extra, what):
    cfg = tmp_path / "cfg.json"
    cfg.write_text(json.dumps({**CFG, **extra}))
    r = subprocess.run([os.path.join(PKG, worker), "--server_info", "", "--cfg_file", str(cfg)],
                       capture_output=True, text=True, timeout=60)
    assert r.returncode == 1 and what in r.stderr, r.stderr


def test_synthetic_mode_refuses_too():
    r = subprocess.run([os.path.join(PKG, "plr_lr_worker"), "--synthetic", "1,10,10,1.0", "--dropout", "0.5"],
                       capture_output=True, text=True, timeout=60)
    assert r.returncode == 1 and "needs storage mxfp4" in r.stderr, r.stderr


@pytest.mark.parametrize("worker", ["plr_lr_worker", "plr_ridge_worker"])
@pytest.mark.parametrize("extra, what", [
    # a rate that rounds to every value dropped: no pass takes it
    ({"storage": "mxfp4", "dropout": 0.999999}, "dropout must be"),
    ({"storage": "mxfp4", "dropout_seed": -5}, "dropout_seed must be"),
    ({"storage": "mxfp4", "dropout_seed": 1 << 64}, "dropout_seed must be")])
def test_values_out_of_range_are_refused(tmp_path, worker, extra, what):
    test_refusals(tmp_path, worker, extra, what)


def test_flags_of_the_synthetic_mode_are_refused_beside_a_cfg_file(tmp_path):
    # a cfg file has keys of these names; a flag beside it was not looked at
    cfg = tmp_path / "cfg.json"
    cfg.write_text(json.dumps(CFG))
    for flag in (["--storage", "mxfp4"], ["--storage=mxfp4", "--dropout=0.5"], ["--dropout_seed", "3"]):
        r = subprocess.run([os.path.join(PKG, "plr_lr_worker"), "--server_info", "", "--cfg_file", str(cfg)] + flag,
                           capture_output=True, text=True, timeout=60)
        assert r.returncode == 1 and "belong to --synthetic" in r.stderr, r.stderr
