"""The arithmetic of oracle/pct_oracle_gelsd.c's BLAS routines is the one that the library's results determine: a few shapes of
tests/golden/derive_blas_orders.py (the whole of it takes a quarter of a minute), and that its probes reject other orders."""
import os
import sys

import numpy as np
import pytest

from oracle import oracle_lib

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden"))
import check_gelsd_port as port  # noqa: E402
import derive_blas_orders as orders  # noqa: E402


@pytest.fixture
def sides():
    try:
        L, core, _ = port.openblas()
    except SystemExit as e:
        pytest.skip(str(e))
    if core not in ("SkylakeX", "Haswell"):
        pytest.skip("NumPy's BLAS runs its %s kernels here" % core)
    O = oracle_lib.lib()
    mode, kernels = oracle_lib.set_lstsq_mode(oracle_lib.LSTSQ_GELSD_AVX2 if core == "Haswell" else oracle_lib.LSTSQ_GELSD), O.gelsd_get_kernel_set()
    O.gelsd_set_kernel_set(1 if core == "Haswell" else 0)
    yield L, O
    oracle_lib.set_lstsq_mode(mode)
    O.gelsd_set_kernel_set(kernels)


def test_sums_have_the_derived_trees(sides):
    lib, G = (sides[0], "library"), (sides[1], "oracle")
    names = ("dgemv T 11 x 7, increment 1", "dgemv T 3 x 2, increment 3", "dgemv T 23 x 7, increment 1", "dgemv N 7 x 11, increment 1",
             "dgemv N 7 x 11, increment 3", "dgemv N 25 x 19, increment 1", "dgemm T N 3 x 3 by 3 x 1", "dgemm T N 25 x 25 by 25 x 1", "dot of 2")
    asked = [k for k in orders.kinds() if k.name in names]
    assert len(asked) == len(names)
    assert orders.check_sums(lib, G, np.random.default_rng(1), asked) == 0
    assert orders.check_elements(lib, G) == 0


def test_norms_are_determined(sides, capsys):
    assert orders.check_dnrm2(*sides, np.random.default_rng(2), (1, 2, 3, 5, 7, 8, 11, 12, 16, 17, 23, 40)) == 0
    assert "join': (((0, 2), 1), 3), 'bits': 64" in capsys.readouterr().out


def test_the_probes_tell_orders_apart():
    """sums of other orders and roundings are found as what they are"""
    def chain(a, x):
        t = 0.0
        for p, q in zip(a, x):
            t = t + p * q
        return np.array([t])

    def pairs(a, x):
        return np.array([(a[0] * x[0] + a[1] * x[1]) + (a[2] * x[2] + a[3] * x[3])])
    found = [orders.text(orders.derive(4, f)[0]) for f in (chain, pairs)]
    assert found == ["(((0 1) 2) 3)", "((0 1) (2 3))"]
    X = orders.near_boundaries(np.random.default_rng(4), 13, 400)  # (13: blocks of 4 and of 8 leave different tails)
    member = dict(w=4, unroll=8, tail="first", join=(((0, 2), 1), 3), bits=64)
    right = np.sqrt(orders.sum_of_squares(X, member)).astype(float)
    for other in (dict(member, bits=53), dict(member, tail="cyclic"), dict(member, join=((0, 1), (2, 3))), dict(member, unroll=4),
                  dict(w=1, unroll=1, tail="first", join=0, bits=64)):
        assert (np.sqrt(orders.sum_of_squares(X, other)).astype(float) != right).sum() > 10
    assert (orders.root_once(orders.sum_of_squares(X, member)) != right).any()
