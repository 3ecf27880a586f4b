"""The bounds of single_term_cases: the six products of pieces keep them in every pass and for
every operand, and no five of them do."""
import numpy as np
import pytest

import single_term_cases as S

CASES = [([130, 5, 0, 129], 96, 200, None), ([40, 0, 200, 31], 2051, 37, 90), ([300], 515, 129, 64),
         ([700, 0, 300, 5], 523, 20, None), ([50, 64, 0, 33] * 2, 1284, 40, 60)]


def _emulated(d, pieces):
    """Every output from products of pieces, with the operands rounded as fp32 rounds them."""
    sq = lambda a: (a * a).astype(np.float32)
    x, v, a = S._rows(d, d["mean"]), S._rows(d, d["var"]), S._rows(d, d["mu_a"])
    out = {}
    for e in range(len(d["offsets"]) - 1):
        r = slice(d["offsets"][e], d["offsets"][e + 1])
        w, q = d["mu_w"][e], d["var_w"][e].astype(np.float64)
        p = lambda y, z: S.product(y, z, pieces)
        parts = dict(mu_z=p(x[r], w), var_z=p(sq(x[r]), d["var_w"][e]), var_only=p(v[r], sq(w)),
                     dz_mu=p(d["row_mu"][r], w.T), dz_var=p(d["row_var"][r], sq(w).T),
                     dw_mu=(q * p(d["column_mu"][r].T, a[r].T))[None],
                     dw_var=(q * q * p(d["column_var"][r].T, sq(a[r]).T))[None])
        for name, value in parts.items():
            out.setdefault(name, []).append(value)
    return {name: np.concatenate(parts) for name, parts in out.items()}


@pytest.mark.parametrize("sizes,K,N,tokens", CASES)
def test_six_products_keep_the_bounds_and_five_do_not(sizes, K, N, tokens):
    d = S.inputs(sizes, K, N, seed=K + N, tokens=tokens)
    want = dict(S.forward(d), **S.state_backward(d), **S.weight_backward(d))
    got = _emulated(d, S.PIECES)
    for name, (value, bound) in want.items():
        assert np.all(np.abs(got[name] - value) <= bound), name
        assert np.count_nonzero(value) > 0
    for left_out in S.PIECES:
        got = _emulated(d, [p for p in S.PIECES if p != left_out])
        for name, (value, bound) in want.items():
            assert np.any(np.abs(got[name] - value) > bound), "%s does without %r" % (name, left_out)
