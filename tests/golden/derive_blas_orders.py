"""The arithmetic of the BLAS routines under np.linalg.lstsq and np.dot, DERIVED from what they return, and compared with
oracle/pct_oracle_gelsd.c (needs the NumPy wheel that bundles OpenBLAS; check_gelsd_port.py says how it is loaded).

Nothing is assumed of a sum but that it adds its products in some binary tree, each addition rounded, a product either rounded
before it is added or fused.  Two probes per pair (i, j) of its terms then determine it:

  * order:   term i = 2^80, term j = -2^80, every other term 1.  Every 1 below the node where i and j meet is lost, every other one
             is kept, so the result is the number of terms outside of the smallest subtree that holds both.  These numbers determine
             the tree (a node is a set of terms whose pairs all meet within it).
  * fusing:  term i = (1 + 2^-30)^2, which is not a float64, term j = -1 times its rounded value, every other term 0.  The result is
             0 unless product i is fused with a partial sum that holds j.

The tree found is evaluated on random vectors against the library (it has to return the same bits: this also tests the assumption)
and compared with the tree that the same probes find in the oracle's routine.

dnrm2 adds squares, which cannot cancel.  Its arithmetic is taken from a family -- 1, 2, 4 or 8 accumulators, any unrolling, four
places for the tail, every order of joining, 53- or 64-bit sums, a root rounded once or twice, scaled sums -- by rejection: vectors
whose sum of squares lies within a few 2^-64 of a rounding boundary of the root, where one different rounding anywhere in the sum
changes the result.  Every member of the family that is left after a few thousand of these has to be the same function as the
oracle's; the others have to be rejected.

    PYTHONDONTWRITEBYTECODE=1 [OPENBLAS_CORETYPE=HASWELL] python tests/golden/derive_blas_orders.py > profiles/blas_orders_<set>.txt
"""
import ctypes as C
import itertools
import math
import os
import sys
from fractions import Fraction

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
import check_gelsd_port as port  # noqa: E402
from check_gelsd_port import D, I, I64, P, dp, fn, ip  # noqa: E402
from oracle import oracle_lib  # noqa: E402

BIG, EPS = 2.0 ** 80, 1.0 + 2.0 ** -30
REST = float(Fraction(EPS) ** 2 - Fraction(EPS * EPS))  # what a fused product keeps
assert REST != 0.0


# ------------------------------------------------------------------------------------------------ the sums: trees of products

def order_probe(terms, i, j):
    """factors (a, x) of a sum of `terms` products, for the pair (i, j)"""
    a, x = np.ones(terms), np.ones(terms)
    a[i], a[j] = BIG, -BIG
    return a, x


def fuse_probe(terms, i, j):
    a, x = np.zeros(terms), np.zeros(terms)
    a[i], x[i] = EPS, EPS
    a[j], x[j] = -(EPS * EPS), 1.0
    return a, x


def derive(terms, sums):
    """`sums(a [terms], x [terms])` -> results of all sums that share these factors.  Their trees, as nested tuples
    (members, left, right), a leaf as (index, fused)"""
    outside, fused = {}, {}
    for i, j in itertools.permutations(range(terms), 2):
        fused[i, j] = sums(*fuse_probe(terms, i, j))
        if i < j:
            outside[i, j] = outside[j, i] = sums(*order_probe(terms, i, j))
    count = len(sums(np.ones(terms), np.ones(terms)))
    trees = []
    for s in range(count):
        size = {p: terms - int(v[s]) for p, v in outside.items()}
        keeps = {p: v[s] for p, v in fused.items()}
        assert all(v in (0.0, REST) for v in keeps.values())
        trees.append(build(tuple(range(terms)), size, keeps))
    return trees


def build(members, size, keeps):
    if len(members) == 1:
        return (members[0], False)
    first = members[0]
    # the two halves of the node: what meets `first` below it, and the rest
    left = tuple(j for j in members if j == first or size[first, j] < len(members))
    right = tuple(j for j in members if j not in left)
    assert right and all(size[i, j] == len(members) for i in left for j in right), "not a tree"
    node = [build(left, size, keeps), build(right, size, keeps)]
    for k, (side, other) in enumerate(((left, right), (right, left))):
        held = {keeps[i, j] != 0.0 for i in side for j in other}
        if True in held:
            assert len(side) == 1 and held == {True}, "a fused product that is not a single term's"
            node[k] = (side[0], True)
    return (members, node[0], node[1])


def evaluate(tree, a, x):
    """(value, exact product or None) of a tree, every rounding as found"""
    if len(tree) == 2:
        return a[tree[0]] * x[tree[0]]
    _, l, r = tree
    for one, other in ((l, r), (r, l)):
        if len(one) == 2 and one[1]:
            v = evaluate(other, a, x)
            exact = Fraction(float(a[one[0]])) * Fraction(float(x[one[0]])) + Fraction(float(v))
            return float(exact)
    return evaluate(l, a, x) + evaluate(r, a, x)


def canonical(tree):
    """the tree with the two sides of every sum in one order (a sum does not depend on it)"""
    if len(tree) == 2:
        return tree
    sides = sorted((canonical(tree[1]), canonical(tree[2])), key=lambda t: min(t[0]) if len(t) == 3 else t[0])
    return (tree[0], sides[0], sides[1])


def text(tree):
    if len(tree) == 2:
        return ("+%d" if tree[1] else "%d") % tree[0]  # "+": fused
    return "(%s %s)" % (text(tree[1]), text(tree[2]))


def gemv(L, trans, alpha, A, x, incx):
    m, n = A.shape
    lda = max(4, m)
    B = np.zeros((lda, n), order="F")
    B[:m] = A
    y = np.zeros(n if trans == "T" else m)
    xs = np.zeros(len(x) * incx)
    xs[::incx] = x
    lib, name = L
    if name == "library":
        fn(lib, "dgemv")(C.c_char_p(trans.encode()), ip(m), ip(n), dp(alpha), P(B), ip(lda), P(xs), ip(incx), dp(0.0), P(y), ip(1), C.c_size_t(1))
    else:
        getattr(lib, "gelsd_dgemv_" + trans.lower())(I(m), I(n), D(alpha), P(B), I(lda), P(xs), I(incx), P(y))
    return y


def gemm(L, V, b):
    """V^T b of an n x n matrix and one column"""
    n = len(b)
    B, c, y = np.asfortranarray(V), b.reshape(n, 1).copy(order="F"), np.zeros((n, 1), order="F")
    lib, name = L
    if name == "library":
        fn(lib, "dgemm")(C.c_char_p(b"T"), C.c_char_p(b"N"), ip(n), ip(1), ip(n), dp(1.0), P(B), ip(n), P(c), ip(n), dp(0.0), P(y), ip(n),
                         C.c_size_t(1), C.c_size_t(1))
    else:
        lib.gelsd_dgemm_tn(I(n), P(B), P(c), P(y))
    return y[:, 0]


def dot2(L, a, x):
    """the products of two 2-vectors that D/space.py:114-115 and :143-145 ask np.dot for"""
    lib, name = L
    if name == "library":
        return np.array([np.dot(a, x)])
    lib.stab_dot2_host.restype = D
    return np.array([lib.stab_dot2_host(D(a[0]), D(a[1]), D(x[0]), D(x[1]))])


class Sums:
    """one kind of call: every result of it is a sum over `terms` products"""
    def __init__(self, name, terms, call, lines):
        self.name, self.terms, self.call, self.lines = name, terms, call, lines

    def shared(self, L):
        """all results at once for factors that every sum shares"""
        def sums(a, x):
            return self.call(L, np.repeat(a[:, None], self.lines, 1), x)
        return sums


def kinds():
    for trans in "TN":
        shapes = [(m, n, s) for m in range(1, 14) for n in range(1, 12) for s in (1, 3)]
        if trans == "T":  # long columns: a 25-supporter system has 301 rows
            shapes += [(m, n, 1) for m in (16, 23, 37, 46, 67) for n in (1, 2, 3, 4, 7)]
        else:
            shapes += [(m, n, 1) for m in (3, 8, 25) for n in (16, 19, 24, 25)] + [(24, 25, 25)]
        for m, n, incx in shapes:
            def call(L, F, x, trans=trans, m=m, n=n, incx=incx):  # F [terms, results]
                return gemv(L, trans, 1.0, F if trans == "T" else F.T, x, incx)
            yield Sums("dgemv %s %d x %d, increment %d" % (trans, m, n, incx), m if trans == "T" else n, call, n if trans == "T" else m)
    for n in range(1, 26):
        yield Sums("dgemm T N %d x %d by %d x 1" % (n, n, n), n, lambda L, F, x: gemm(L, F, x), n)
    yield Sums("dot of 2", 2, lambda L, F, x: dot2(L, np.ascontiguousarray(F[:, 0]), x), 1)


def check_sums(lib, G, rng, asked=None):
    bad = 0
    seen = {}
    for kind in asked or kinds():
        found = derive(kind.terms, kind.shared(lib)) if kind.terms > 1 else None
        if found is not None:
            mine = derive(kind.terms, kind.shared(G))
            if [canonical(t) for t in found] != [canonical(t) for t in mine]:
                bad += 1
                print("%s: library %s, oracle %s" % (kind.name, [text(t) for t in found], [text(t) for t in mine]))
        for _ in range(3):
            F, x = rng.standard_normal((kind.terms, kind.lines)), rng.standard_normal(kind.terms)
            got, other = kind.call(lib, F, x), kind.call(G, F, x)
            want = np.array([evaluate(t, F[:, s], x) for s, t in enumerate(found)]) if found is not None else F[0] * x[0]
            if not (np.array_equal(got, want) and np.array_equal(got, other)):
                bad += 1
                print("%s: random vectors differ (tree %s, oracle %s)" % (kind.name, np.array_equal(got, want), np.array_equal(got, other)))
        if found is not None:
            seen.setdefault(kind.name.split(" ")[0], []).append((kind.name, [text(t) for t in found]))
    for key, shows in seen.items():
        print("%s: %d shapes derived" % (key, len(shows)))
    for name in ("dgemv T 11 x 7, increment 1", "dgemv N 7 x 11, increment 1", "dgemv N 7 x 11, increment 3", "dgemm T N 13 x 13 by 13 x 1", "dot of 2"):
        for n, trees in seen.get(name.split(" ")[0], ()):
            if n == name:
                print("  %s (numbers: terms in order; +: the product is fused into the sum beside it)" % n)
                for s, t in enumerate(trees):
                    print("    result %2d: %s" % (s, t))
    return bad


def check_alpha(lib, G):
    """a factor before a sum: dgemv's products of alpha with x or with a block's sum, dger's alpha y"""
    bad = 0
    rng = np.random.default_rng(3)
    for trans in "TN":
        for m in range(1, 14):
            for n in range(1, 12):
                k = m if trans == "T" else n
                for i in range(k):
                    for j in range(k):
                        t = np.zeros(k)
                        t[i], t[j] = EPS, (0.0 if i == j else -EPS)
                        x = np.ones(k)
                        A = np.repeat(t[:, None], n, 1) if trans == "T" else np.repeat(t[None], m, 0)
                        bad += not np.array_equal(gemv(lib, trans, EPS, A, x, 1), gemv(G, trans, EPS, A, x, 1))
                A, x = rng.standard_normal((m, n)), rng.standard_normal(k)
                bad += not np.array_equal(gemv(lib, trans, -0.7, A, x, 1), gemv(G, trans, -0.7, A, x, 1))
    print("dgemv with alpha not 1: %d calls differ" % bad)
    return bad


def check_elements(lib, G):
    """dger and drot: which product of an element's is fused, and which pair of dger's three factors is multiplied first"""
    bad = 0
    L, O = lib[0], G[0]
    e2 = EPS * EPS
    for m in list(range(1, 41)) + [63, 64, 65, 300]:
        res = []
        for alpha, yv, xv, a in ((1.0, EPS, EPS, -e2), (EPS, EPS, 1.0, -e2), (EPS, 1.0, EPS, -e2)):
            pair = []
            for which in (0, 1):
                A, x, y = np.asfortranarray(np.full((max(4, m), 1), a)), np.full(m, xv), np.full(1, yv)
                if which:
                    O.gelsd_dger(I(m), I(1), D(alpha), P(x), I(1), P(y), I(1), P(A), I(max(4, m)))
                else:
                    fn(L, "dger")(ip(m), ip(1), dp(alpha), P(x), ip(1), P(y), ip(1), P(A), ip(max(4, m)))
                pair.append(A[:m, 0])
            bad += not np.array_equal(*pair)
            res.append(pair[0])
        first, second, third = ([int(v != 0.0) for v in r] for r in res)
        if m in (16, 23):
            print("  dger, %d elements: fused %s; alpha y rounded first %s; alpha x rounded first %s" %
                  (m, "".join(map(str, first)), not any(second), not any(third)))
        for u, v, c, s in ((EPS, -e2, EPS, 1.0), (1.0, EPS, -e2, EPS), (e2, EPS, EPS, 1.0), (EPS, e2, 1.0, EPS)):
            pair = []
            for which in (0, 1):
                p, q = np.full(m, u), np.full(m, v)
                if which:
                    O.gelsd_drot(I(m), P(p), I(1), P(q), I(1), D(c), D(s))
                else:
                    fn(L, "drot")(ip(m), P(p), ip(1), P(q), ip(1), dp(c), dp(s))
                pair.append(np.concatenate([p, q]))
            bad += not np.array_equal(*pair)
            if m == 7:
                print("  drot x = %g, y = %g, c = %g, s = %g: c x + s y keeps %s, c y - s x keeps %s" % (u, v, c, s, pair[0][0], pair[0][m]))
    print("dger, drot: %d calls differ" % bad)
    return bad


# ---------------------------------------------------------------------------------------------------------------------- dnrm2

def trees_over(leaves):
    """every order of joining labelled partial sums"""
    if len(leaves) == 1:
        yield leaves[0]
        return
    first, rest = leaves[0], leaves[1:]
    for k in range(len(rest)):
        for with_first in itertools.combinations(rest, k):
            left = (first,) + with_first
            right = tuple(x for x in rest if x not in with_first)
            for l in trees_over(left):
                for r in trees_over(right):
                    yield (l, r)


def joins(w):
    if w <= 4:
        return list(trees_over(tuple(range(w))))
    chain, pair = 0, [0, 1, 2, 3, 4, 5, 6, 7]
    for k in range(1, 8):
        chain = (chain, k)
    far = [(k, k + 4) for k in range(4)]
    while len(pair) > 1:
        pair = [(pair[k], pair[k + 1]) for k in range(0, len(pair), 2)]
    return [chain, pair[0], (((far[0], far[2]), (far[1], far[3]))), (((far[0], far[1]), (far[2], far[3])))]


def family():
    for w in (1, 2, 4, 8):
        for unroll in sorted({w, 2 * w, 4 * w, 8, 16}):
            if unroll % w or (w == 1 and unroll > 1):
                continue
            for tail in (("first", "last", "cyclic", "after") if w > 1 else ("first",)):
                for join in joins(w):
                    for bits in (64, 53):
                        yield dict(w=w, unroll=unroll, tail=tail, join=join, bits=bits)


def sum_of_squares(X, f):
    """the rows' sums of squares by member f of the family"""
    kind = np.longdouble if f["bits"] == 64 else np.float64
    Y = X.astype(kind)
    S = Y * Y
    n, w = X.shape[1], f["w"]
    lead = n - n % f["unroll"]
    acc = [np.zeros(len(X), kind) for _ in range(w)]
    after = []
    for i in range(n):
        if i < lead or f["tail"] == "cyclic":
            acc[i % w] = acc[i % w] + S[:, i]
        elif f["tail"] == "first":
            acc[0] = acc[0] + S[:, i]
        elif f["tail"] == "last":
            acc[w - 1] = acc[w - 1] + S[:, i]
        else:
            after.append(S[:, i])

    def join(t):
        return acc[t] if isinstance(t, int) else join(t[0]) + join(t[1])
    total = join(f["join"])
    for t in after:
        total = total + t
    return total


def root_once(total):
    """the square roots of 64-bit sums rounded to a double in one step"""
    out = []
    for t in total:
        m, e = math.frexp(t) if isinstance(t, float) else np.frexp(t)
        num = int(np.ldexp(m, 64))
        e = int(e) - 64
        if e & 1:
            num, e = num * 2, e - 1
        s = math.isqrt(num << 160)  # 2^80 sqrt(num), cut: a sticky bit stands in for the rest
        s = s * 2 + (s * s != num << 160)
        out.append(float(Fraction(s) * Fraction(2) ** (e // 2 - 81)))
    return np.array(out)


def near_boundaries(rng, n, count):
    """vectors of n elements whose sum of squares is within a few 2^-64 of the square of a midpoint between two doubles"""
    X = np.zeros((count, n))
    for r in range(count):
        x = rng.standard_normal(n) * 2.0 ** rng.integers(-2, 3, n)
        if n > 1:
            k = int(rng.integers(0, n))
            rest = sum((Fraction(float(v)) ** 2 for i, v in enumerate(x) if i != k), Fraction(0))
            # element k is about 2^-6 of the norm, so that a step of it moves the sum by less than 2^-64
            norm = Fraction(math.sqrt(float(rest)) * (1 + 2.0 ** -13))
            mid = Fraction(float(norm)) + Fraction(math.ulp(float(norm))) / 2
            need = mid * mid - rest + Fraction(int(rng.integers(-6, 7)), 2 ** 65) * mid * mid
            x[k] = math.sqrt(float(need)) if need > 0 else x[k]
            if need > 0:  # the double whose square is nearest
                x[k] = min((x[k], np.nextafter(x[k], 0), np.nextafter(x[k], 9e9)), key=lambda v: abs(Fraction(float(v)) ** 2 - need))
        X[r] = x
    return X


def check_dnrm2(L, O, rng, sizes=tuple(range(1, 41)) + (48, 64, 67, 100, 130, 191, 300)):
    nrm = L.scipy_cblas_dnrm264_
    nrm.restype = D
    O.gelsd_dnrm2.restype = D
    alive, why = list(family()), {}
    full = len(alive)
    bad = calls = twice_only = 0
    for n in sizes:
        X = near_boundaries(rng, n, 400 if n <= 40 else 120)
        got = np.array([nrm(I64(n), P(v), I64(1)) for v in X])
        mine = np.array([O.gelsd_dnrm2(I(n), P(v), I(1)) for v in X])
        calls += len(X)
        bad += int((got != mine).sum())
        spread = np.array([nrm(I64(n), P(np.ascontiguousarray(np.repeat(v, 3))), I64(3)) for v in X[:50]])
        bad += int((spread != got[:50]).sum())
        left = []
        for f in alive:
            total = sum_of_squares(X, f)
            if np.array_equal(np.sqrt(total).astype(np.float64), got):
                left.append(f)
            else:
                why[(f["w"], f["bits"])] = why.get((f["w"], f["bits"]), 0) + 1
        alive = left
        if n in (5, 8, 12, 17, 40):
            once = root_once(sum_of_squares(X, dict(w=4, unroll=8, tail="first", join=(((2, 0), 1), 3), bits=64)))
            twice_only += int((once != got).sum())
    print("dnrm2: %d calls near a rounding boundary, oracle differs on %d" % (calls, bad))
    print("  members of the family: %d, rejected (accumulators, bits): %s, left:" % (full, why))
    for f in alive:
        print("   ", f)
    print("  root rounded to a double in one step instead of through 64 bits: %d results would differ" % twice_only)
    # what is left has to be one function: the sum's order, its precision and the tail's place
    same = {(f["w"], f["unroll"], f["tail"], str(f["join"]), f["bits"]) for f in alive}
    if len(same) != 1 or not twice_only:
        print("  dnrm2 is NOT determined by these outputs")
        bad += 1
    return bad


def main():
    L, core, cfg = port.openblas()
    O = oracle_lib.lib()
    oracle_lib.set_lstsq_mode(oracle_lib.LSTSQ_GELSD_AVX2 if core == "Haswell" else oracle_lib.LSTSQ_GELSD)
    O.gelsd_set_kernel_set(I(1 if core == "Haswell" else 0))
    rng = np.random.default_rng(11)
    print("NumPy %s, %s, kernel set %s" % (np.__version__, cfg.strip(), core))
    lib, G = (L, "library"), (O, "oracle")
    bad = check_sums(lib, G, rng) + check_alpha(lib, G) + check_elements(lib, G) + check_dnrm2(L, O, rng)
    print("TOTAL differences: %d" % bad)
    return 1 if bad else 0


if __name__ == "__main__":
    sys.exit(main())
