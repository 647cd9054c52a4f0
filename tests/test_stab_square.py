"""CPU: the lever rule's square as it ships (csrc/pct_stab.cuh lever_square: len * len), compiled for the host, and what it does to
verdicts where the reference's power, the C library's pow(len, 2.0), has another last bit."""
import ctypes

import numpy as np

import oracle.oracle_lib as ol
from tests.common import item_set_range, make_stream
from tests.test_stab_host import VARIANT, _Variant


def test_the_host_build_runs_the_square_that_ships():
    with _Variant():
        var = ctypes.CDLL(VARIANT)
    f = var.stab_host_lever_square
    f.restype, f.argtypes = ctypes.c_double, [ctypes.c_double]
    var.pow_host.restype, var.pow_host.argtypes = ctypes.c_double, [ctypes.c_double] * 2
    rng = np.random.default_rng(6)
    lens = np.sqrt(rng.integers(1, 10 ** 12, 200000) * 2.5e-13)
    assert [f(x) for x in lens.tolist()] == (lens * lens).tolist()
    var.stab_host_set_pow(1)
    try:
        assert [f(x) for x in lens[:5000].tolist()] == [var.pow_host(x, 2.0) for x in lens[:5000].tolist()]
    finally:
        var.stab_host_set_pow(0)
    out = (ctypes.c_long * 3)()
    var.pow_host_sweep_continuous(ctypes.c_long(2_000_000), ctypes.c_ulonglong(5), ctypes.c_double(1.0), out)
    assert out[1] == 0 and 0.0005 < out[2] / out[0] < 0.0011, tuple(out)  # every one correctly rounded; the power differs on 0.08 %


def _run(make, stream, steps, square=None):
    var = ctypes.CDLL(VARIANT)
    if square is not None:
        var.stab_host_set_pow(square)
    try:
        env = make()
        env.set_item_stream(stream)
        env.reset()
        obs, done = [], []
        for _ in range(steps):
            obs.append(env.obs.copy())
            env.step_hash_policy(1)
            done.append(env.done.copy())
        env.close()
    finally:
        var.stab_host_set_pow(0)
    return np.array(obs), np.array(done)


def test_verdicts_with_the_square_and_with_the_power():
    """the product's stability source with the power is the oracle, observation for observation; with the square that ships an
    env may part ways at a verdict that hangs on the last bit: none of these does"""
    rng = np.random.default_rng(12)
    unit = lambda: ol.OracleVecEnv(24, setting=1, container_size=(1, 1, 1), env_kind=1, sample_bounds=(0.1, 0.5), internal_node_holder=80, leaf_node_holder=50)
    items = item_set_range(5, 30)[::97]
    large = lambda: ol.OracleVecEnv(24, setting=1, container_size=(60, 60, 60), item_set=items, internal_node_holder=80, leaf_node_holder=50)
    for make, stream, steps in ((unit, rng.integers(100, 501, (24, 512, 3)).astype(np.int32), 250), (large, make_stream(3, 24, 512, items), 250)):
        env = make()
        env.set_item_stream(stream)
        env.reset()
        obs, done = [], []
        for _ in range(steps):
            obs.append(env.obs.copy())
            env.step_hash_policy(1)
            done.append(env.done.copy())
        env.close()
        with _Variant():
            power = _run(make, stream, steps, 1)
            square = _run(make, stream, steps, 0)
        assert np.array_equal(power[0], obs) and np.array_equal(power[1], done)
        parted = [e for e in range(24) if not np.array_equal(square[0][:, e], power[0][:, e])]
        assert not parted
        assert np.array(done).sum() > 24  # (episodes end: verdicts were met)
