"""In which order the BLAS routines under np.linalg.lstsq add, and what they fuse, read off their OUTPUTS -- and whether
oracle/pct_oracle_gelsd.c does the same (needs the NumPy wheel that bundles OpenBLAS; see check_gelsd_port.py for the loading).

Two probes per pair (i, j) of the terms of one sum, everything else chosen so that the exact result is known:

  * order:  term i = 2^80, term j = -2^80, every other term 1.  A 1 that is added to a partial sum holding only one of the two is
            lost, one that joins after they met is kept, so the result counts the terms outside the smallest subtree of the
            summation tree that holds i and j.  The counts of all pairs determine the tree.
  * fusing: term i = (1 + 2^-30)^2, not a float64, term j = -1 times its rounded value, every other term 0.  The result is 0
            where the product was rounded before it was added, else its rounding error (with a sign that says which of the two).

Both are taken of the library's routine and of the restatement for every shape up to the sizes below and compared entry by entry.
dnrm2 adds squares, which cannot cancel; the probes of it here compare results only, and other orders return the same ones.  What
determines its order, dgemm's and np.dot's is derive_blas_orders.py.

    PYTHONDONTWRITEBYTECODE=1 python tests/golden/check_blas_order.py
"""
import ctypes as C
import os
import sys

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
import check_gelsd_port as port  # noqa: E402
from check_gelsd_port import D, I, I64, P, dp, fn, ip  # noqa: E402
from oracle import oracle_lib  # noqa: E402

BIG, EPS = 2.0 ** 80, 1.0 + 2.0 ** -30


def gemv(L, trans, A, x, incx):
    m, n = A.shape
    lda = max(4, m)
    B = np.zeros((lda, n), order="F")
    B[:m] = A
    y = np.zeros(n if trans == "T" else m)
    xs = np.zeros(len(x) * incx)
    xs[::incx] = x
    lib, name = L
    if name == "library":
        fn(lib, "dgemv")(C.c_char_p(trans.encode()), ip(m), ip(n), dp(1.0), P(B), ip(lda), P(xs), ip(incx), dp(0.0), P(y), ip(1), C.c_size_t(1))
    else:
        getattr(lib, "gelsd_dgemv_" + trans.lower())(I(m), I(n), D(1.0), P(B), I(lda), P(xs), I(incx), P(y))
    return y


def probes(L, trans, m, n, incx):
    """for every pair of terms: the counts and the rounding errors of every element of the result"""
    k = m if trans == "T" else n
    out = []
    for i in range(k):
        for j in range(k):
            if i == j:
                continue
            x = np.ones(k)
            A = np.ones((m, n))
            t = A if trans == "T" else A.T  # t[term] = the factors of that term in every sum
            t[i], t[j] = BIG, -BIG
            out.append(gemv(L, trans, A, x, incx))
            A = np.zeros((m, n))
            t = A if trans == "T" else A.T
            x = np.zeros(k)
            t[i], x[i] = EPS, EPS
            t[j], x[j] = -(EPS * EPS), 1.0
            out.append(gemv(L, trans, A, x, incx))
    return np.array(out) if out else np.zeros((0, n if trans == "T" else m))


def norms(L, n):
    out = []
    for i in range(n):
        x = np.full(n, 2.0 ** -33)  # squares of 2^-66: against 1 each is lost in 80 bits, 8 of them together are not
        x[i] = 1.0
        out.append(L(n, x))
        x = np.full(n, 1.0 + 2.0 ** -31)
        x[i] = 2.0 ** 31 + 1.0
        out.append(L(n, x))
    return np.array(out)


def main():
    lib, core, cfg = port.openblas()
    G = oracle_lib.lib()
    G.gelsd_set_kernel_set(I(1 if core.lower() in ("haswell", "zen") else 0))
    print("NumPy %s, %s, kernel set %s" % (np.__version__, cfg.strip(), core))
    bad = shapes = 0
    for trans in "TN":
        for m in range(1, 14):
            for n in range(1, 12):
                for incx in (1, 3):
                    a, b = (probes(l, trans, m, n, incx) for l in ((lib, "library"), (G, "oracle")))
                    shapes += 1
                    if not np.array_equal(a, b):
                        bad += 1
                        print("dgemv %s %d x %d, increment %d: %d of %d probes differ" % (trans, m, n, incx, (a != b).any(1).sum(), len(a)))
    nrm = lib.scipy_cblas_dnrm264_
    nrm.restype = D
    G.gelsd_dnrm2.restype = D
    for n in range(1, 41):
        shapes += 1
        a, b = norms(lambda k, x: nrm(I64(k), P(x), I64(1)), n), norms(lambda k, x: G.gelsd_dnrm2(I(k), P(x), I(1)), n)
        if not np.array_equal(a, b):
            bad += 1
            print("dnrm2 %d: %d of %d probes differ" % (n, (a != b).sum(), len(a)))
    # dger and drot: one product and one sum (two products) to an element -- which products are fused, element by element
    for m in range(1, 41):
        shapes += 1
        res = []
        for which in ("library", "oracle"):
            A = np.asfortranarray(np.full((max(4, m), 1), -(EPS * EPS)))
            x, y = np.full(m, EPS), np.full(1, EPS)
            if which == "library":
                fn(lib, "dger")(ip(m), ip(1), dp(1.0), P(x), ip(1), P(y), ip(1), P(A), ip(max(4, m)))
            else:
                G.gelsd_dger(I(m), I(1), D(1.0), P(x), I(1), P(y), I(1), P(A), I(max(4, m)))
            rot = []
            for u, v, c, s in ((EPS, -(EPS * EPS), EPS, 1.0), (1.0, EPS, -(EPS * EPS), EPS), (EPS * EPS, EPS, EPS, 1.0), (EPS, EPS * EPS, 1.0, EPS)):
                p, q = np.full(m, u), np.full(m, v)
                if which == "library":
                    fn(lib, "drot")(ip(m), P(p), ip(1), P(q), ip(1), dp(c), dp(s))
                else:
                    G.gelsd_drot(I(m), P(p), I(1), P(q), I(1), D(c), D(s))
                rot += [p, q]
            res.append(np.concatenate([A[:m, 0]] + rot))
        if not np.array_equal(*res):
            bad += 1
            print("dger / drot of %d: %d elements differ" % (m, (res[0] != res[1]).sum()))
    print("%d shapes probed, %d differ" % (shapes, bad))
    return 1 if bad else 0


if __name__ == "__main__":
    raise SystemExit(main())
