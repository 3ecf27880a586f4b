"""Expert-grouped Linear layers on sums of a single term: activations (or innovations) with one
number other than zero in every reduction, so that an output is one product of two fp32 numbers
and its error that of the product alone, however long the reduction is.

The matrix kernels take a number apart into three bf16 pieces h + m + l and form hh, hm, mh, mm,
hl and lh of two of them, the smallest first. What they leave out (ml, lm, ll and what the pieces
do not hold) is at most 2^-25 of the product, U / 2 with U = 2^-24. Products of two pieces are
exact; each of the six additions rounds by at most U of the product. Zeros add nothing. That
makes 6.5 U; a factor that is itself a rounded square, and every multiplication behind the sum,
adds U. A piece product that is missing shows: mm, hl and lh are up to 2^-18 of the product, 64 U.
"""
import numpy as np

import moe_cases as C

PRODUCT = 6.5      # in U


def inputs(sizes, K, N, seed, tokens=None):
    """d: as moe_cases.grouped_inputs, with mu_a, var_a, dmu and dvar as `mean`, `var`, `row` and
    `column` below replace them."""
    d = C.grouped_inputs(sizes, K, N, seed=seed, tokens=tokens)
    rng = np.random.default_rng(seed + 1)
    held, R = d["mu_a"].shape[0], int(d["offsets"][-1])

    def one_per_row(a, width):
        """a with all but one element of every row zero; the places walk through all columns"""
        out = np.zeros_like(a)
        at = (np.arange(a.shape[0]) * 37 + 11) % width
        out[np.arange(a.shape[0]), at] = a[np.arange(a.shape[0]), at]
        return out

    def one_per_column(a):
        """the same for the columns of every expert's rows"""
        out = np.zeros_like(a)
        for e in range(len(sizes)):
            first, rows = d["offsets"][e], sizes[e]
            if rows:
                at = first + (np.arange(N) * 13 + 5) % rows
                out[at, np.arange(N)] = a[at, np.arange(N)]
        return out
    mu, var = d["mu_a"], rng.uniform(0.1, 1, (held, K)).astype(np.float32)
    d["mean"], d["var"] = one_per_row(mu, K), one_per_row(var, K)
    d["row_mu"], d["row_var"] = one_per_row(d["dmu"][:R], N), one_per_row(d["dvar"][:R], N)
    d["column_mu"], d["column_var"] = one_per_column(d["dmu"][:R]), one_per_column(d["dvar"][:R])
    return d


def _by_expert(d, call):
    """{name: (value, bound)} of all rows (or experts) from call(e, rows of expert e)."""
    out = {}
    for e in range(len(d["offsets"]) - 1):
        r = slice(d["offsets"][e], d["offsets"][e + 1])
        for name, (value, c) in call(e, r).items():
            out.setdefault(name, []).append((value, 1.001 * c * C.U * np.abs(value)))
    return {name: tuple(np.concatenate([p[i] for p in parts]) for i in range(2)) for name, parts in out.items()}


def _rows(d, a):
    return a if d["rows"] is None else a[d["rows"]]


def forward(d):
    """mu_z and var_z of (mean, 0), and var_z of (0, var) with weights of no variance."""
    x, v = _rows(d, d["mean"]).astype(np.float64), _rows(d, d["var"]).astype(np.float64)
    mw, vw = d["mu_w"].astype(np.float64), d["var_w"].astype(np.float64)
    return _by_expert(d, lambda e, r: dict(
        mu_z=(x[r] @ mw[e].T, PRODUCT), var_z=(x[r] ** 2 @ vw[e].T, PRODUCT + 1),
        var_only=(v[r] @ (mw[e] ** 2).T, PRODUCT + 1)))


def state_backward(d):
    m, v = d["row_mu"].astype(np.float64), d["row_var"].astype(np.float64)
    mw = d["mu_w"].astype(np.float64)
    return _by_expert(d, lambda e, r: dict(dz_mu=(m[r] @ mw[e], PRODUCT), dz_var=(v[r] @ mw[e] ** 2, PRODUCT + 1)))


def weight_backward(d):
    a = _rows(d, d["mu_a"]).astype(np.float64)
    m, v = d["column_mu"].astype(np.float64), d["column_var"].astype(np.float64)
    q = d["var_w"].astype(np.float64)
    return _by_expert(d, lambda e, r: dict(
        dw_mu=((q[e] * (m[r].T @ a[r]))[None], PRODUCT + 1),
        dw_var=((q[e] ** 2 * (v[r].T @ a[r] ** 2))[None], PRODUCT + 3)))


# ---- the products of pieces, on the CPU ---------------------------------------------------------

PIECES = [(0, 0), (0, 1), (1, 0), (1, 1), (0, 2), (2, 0)]


def split(x):
    """The three bf16 pieces of fp32 numbers, each rounded to nearest even, in 64 bits."""
    out, rest = [], np.asarray(x, np.float32)
    for _ in range(3):
        u = rest.view(np.uint32).astype(np.uint64)
        u = ((u + 0x7fff + ((u >> 16) & 1)) >> 16) << 16
        piece = u.astype(np.uint32).view(np.float32)
        out.append(piece.astype(np.float64))
        rest = rest - piece
    return out


def product(x, y, pieces=PIECES):
    """Matrix product x y^T (fp32, fp32) from the given pairs of pieces."""
    a, b = split(x), split(y)
    return sum(a[i] @ b[j].T for i, j in pieces)
