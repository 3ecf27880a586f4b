"""Layer norm, expert-grouped Linear layers and the mixture-of-experts router: seeded
inputs, the operators in 64 bits, and error bounds derived from the arithmetic.

The 64-bit forms are plain numpy. Every bound is an absolute one per element, a count of
roundings times U times the sum of the magnitudes of the terms that were added: a sum of S
terms in any order, each the product of rounded factors, is off by at most (S + c) * U *
sum|terms|, U = 2^-24 half a step of fp32, c the roundings of a term's own factors. The
matrix kernels form a product of two fp32 numbers from up to six products of 8-bit pieces
that the accumulator takes one after the other, hence 6 S instead of S; what they leave out
of a product is below 2^-25 of it, inside c.
"""
import numpy as np

U = 2.0 ** -24


def check(got, want, bound, what):
    got = np.asarray(got, np.float64)
    want, bound = np.asarray(want, np.float64), np.asarray(bound, np.float64)
    assert got.shape == want.shape, "%s: shape %s, expected %s" % (what, got.shape, want.shape)
    assert np.all(np.isfinite(got)), what + ": non-finite values"
    over = np.abs(got - want) - (bound + 1e-37)
    if got.size and over.max() > 0:
        at = np.unravel_index(np.argmax(over), over.shape)
        raise AssertionError("%s%s: %r, expected %r, bound %.3e" % (what, at, got[at], want[at],
                                                                   np.broadcast_to(bound, want.shape)[at]))


# ---- layer norm ------------------------------------------------------------------------

def norm_inputs(B, n, seed=0, shift=1.0):
    rng = np.random.default_rng(seed)
    f = np.float32
    return dict(
        mu_w=(1 + 0.1 * rng.standard_normal(n)).astype(f), var_w=rng.uniform(0.01, 0.1, n).astype(f),
        mu_b=(0.1 * rng.standard_normal(n)).astype(f), var_b=rng.uniform(0.01, 0.1, n).astype(f),
        mu_a=(rng.standard_normal((B, n)) + shift * rng.standard_normal((B, 1))).astype(f),
        var_a=rng.uniform(0.01, 0.5, (B, n)).astype(f), jcb=rng.uniform(0, 1, (B, n)).astype(f),
        dmu=(0.1 * rng.standard_normal((B, n))).astype(f),
        dvar=(-rng.uniform(0, 1e-2, (B, n))).astype(f))


def norm_fwd(d, eps, bias=True):
    """{name: (value, bound)} of mu_z, var_z, mu_s, var_s."""
    a, v = d["mu_a"].astype(np.float64), d["var_a"].astype(np.float64)
    mw, vw = d["mu_w"].astype(np.float64), d["var_w"].astype(np.float64)
    n = a.shape[1]
    mean = a.mean(1)
    e_mean = (n + 2) * U * np.abs(a).mean(1)
    c = a - mean[:, None]
    e_c = e_mean[:, None] + U * np.abs(c)
    total = (c * c).sum(1) + v.sum(1)
    var = total / (n - 1)
    # the squares carry twice the deviation's error, the sum its n + 4 roundings
    e_var = ((n + 4) * U * total + (2 * np.abs(c) * e_c + e_c * e_c).sum(1)) / (n - 1)
    inv = 1 / np.sqrt(var + eps)
    r_inv = (0.5 * e_var / (var + eps) + 4 * U)[:, None]          # relative, sqrt and division
    inv = inv[:, None]
    x = inv * c
    e_x = np.abs(x) * (r_inv + 2 * U) + inv * e_c
    mu_z, e_mu = x * mw, (e_x + U * np.abs(x)) * np.abs(mw)
    s = inv * inv * v * (mw * mw + vw)
    q = vw * x * x
    var_z, e_v = s + q, s * (2 * r_inv + 6 * U) + vw * (2 * np.abs(x) * e_x + e_x * e_x) + q * 4 * U
    e_v = e_v + U * var_z
    if bias:
        mb, vb = d["mu_b"].astype(np.float64), d["var_b"].astype(np.float64)
        mu_z, var_z = mu_z + mb, var_z + vb
        e_mu, e_v = e_mu + U * np.abs(mu_z), e_v + U * var_z
    return dict(mu_z=(mu_z, 1.01 * e_mu), var_z=(var_z, 1.01 * e_v), mu_s=(mean, 1.01 * e_mean),
                var_s=(var, 1.01 * e_var))


def norm_bwd(d, mu_s, var_s, eps, jcb=True):
    """Of the six innovations; mu_s / var_s are the fp32 statistics that the call was given."""
    g = {k: x.astype(np.float64) for k, x in d.items()}
    B, n = g["dmu"].shape
    mean, inv = mu_s.astype(np.float64)[:, None], 1 / np.sqrt(var_s.astype(np.float64) + eps)[:, None]
    t = inv * g["mu_w"] * (g["jcb"] if jcb else 1.0)
    x = inv * (g["mu_a"] - mean)
    dm, dv = g["dmu"], g["dvar"]
    # inv: sum, root and quotient, 3 U (the sum's error halves under the root); the factors and
    # the products of a term: at most 8 U (mean), 14 U (variance, where inv and x enter twice)
    out = dict(dz_mu=(t * dm, 8 * U * np.abs(t * dm)), dz_var=(t * t * dv, 14 * U * np.abs(t * t * dv)))
    vw, vb = g["var_w"], g["var_b"]

    def column(name, terms, factor, c):
        out[name] = (factor * terms.sum(0), 1.01 * (B + c) * U * factor * np.abs(terms).sum(0))
    column("dw_mu", x * dm, vw, 10)
    column("dw_var", x * x * dv, vw * vw, 18)
    column("db_mu", dm, vb, 3)
    column("db_var", dv, vb * vb, 4)
    return out


# ---- grouped Linear ----------------------------------------------------------------------

def grouped_inputs(sizes, K, N, seed=0, tokens=None, tail=0):
    """sizes: rows of every expert. tokens: the rows come from that many tokens. tail: rows
    behind the last group."""
    rng = np.random.default_rng(seed)
    f = np.float32
    E, R = len(sizes), int(sum(sizes)) + tail
    held = R if tokens is None else tokens
    d = dict(
        mu_w=rng.normal(0, K ** -0.5, (E, N, K)).astype(f),
        var_w=(rng.uniform(0.5, 1.5, (E, N, K)) / K).astype(f),
        mu_b=rng.normal(0, 0.5, (E, N)).astype(f), var_b=(rng.uniform(0.5, 1.5, (E, N)) / K).astype(f),
        mu_a=rng.normal(0, 1, (held, K)).astype(f), var_a=rng.uniform(0.01, 0.1, (held, K)).astype(f),
        jcb=rng.uniform(0, 1, (R, K)).astype(f), dmu=rng.normal(0, 0.1, (R, N)).astype(f),
        dvar=(-rng.uniform(0, 1e-3, (R, N))).astype(f))
    d["offsets"] = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    d["rows"] = None if tokens is None else rng.integers(0, tokens, R).astype(np.int32)
    return d


def _held(d, name):
    """Activations row by row; an index outside the tokens stands for zeros."""
    a = d[name].astype(np.float64)
    if d["rows"] is None:
        return a
    ok = (d["rows"] >= 0) & (d["rows"] < a.shape[0])
    return np.where(ok[:, None], a[np.where(ok, d["rows"], 0)], 0.0)


def grouped_fwd(d, bias=True):
    """(value, bound) of mu_z, var_z over the rows of the groups."""
    x, v = _held(d, "mu_a"), _held(d, "var_a")
    mw, vw = d["mu_w"].astype(np.float64), d["var_w"].astype(np.float64)
    E, N, K = mw.shape
    R = d["offsets"][-1]
    z = {k: np.zeros((R, N)) for k in ("mu_z", "var_z", "e_mu", "e_var")}
    for e in range(E):
        r = slice(d["offsets"][e], d["offsets"][e + 1])
        z["mu_z"][r] = x[r] @ mw[e].T
        z["e_mu"][r] = (6 * K + 16) * U * (np.abs(x[r]) @ np.abs(mw[e]).T)
        z["var_z"][r] = (v[r] + x[r] ** 2) @ vw[e].T + v[r] @ (mw[e] ** 2).T
        z["e_var"][r] = (12 * K + 16) * U * z["var_z"][r]
        if bias:
            mb, vb = d["mu_b"][e].astype(np.float64), d["var_b"][e].astype(np.float64)
            z["e_mu"][r] += 2 * U * np.abs(mb)
            z["e_var"][r] += 2 * U * vb
            z["mu_z"][r] += mb
            z["var_z"][r] += vb
    return dict(mu_z=(z["mu_z"], z["e_mu"]), var_z=(z["var_z"], z["e_var"]))


def grouped_bwd(d, jcb=True):
    x = _held(d, "mu_a")
    g = {k: d[k].astype(np.float64) for k in ("mu_w", "var_w", "var_b", "jcb", "dmu", "dvar")}
    E, N, K = g["mu_w"].shape
    R = d["offsets"][-1]
    out = {}

    def put(name, at, shape, value, magnitude, c):
        v, b = out.setdefault(name, (np.zeros(shape), np.zeros(shape)))
        v[at] = value
        b[at] = 1.01 * c * U * magnitude
    for e in range(E):
        r = slice(d["offsets"][e], d["offsets"][e + 1])
        S = d["offsets"][e + 1] - d["offsets"][e]
        j = g["jcb"][r] if jcb else 1.0
        dm, dv, w, q = g["dmu"][r], g["dvar"][r], g["mu_w"][e], g["var_w"][e]
        put("dz_mu", r, (R, K), j * (dm @ w), j * (np.abs(dm) @ np.abs(w)), 6 * N + 16)
        put("dz_var", r, (R, K), j * j * (dv @ w ** 2), j * j * (np.abs(dv) @ w ** 2), 6 * N + 16)
        put("dw_mu", e, (E, N, K), q * (dm.T @ x[r]), q * (np.abs(dm).T @ np.abs(x[r])), 6 * S + 16)
        put("dw_var", e, (E, N, K), q * q * (dv.T @ x[r] ** 2), q * q * (np.abs(dv).T @ x[r] ** 2), 6 * S + 16)
        vb = g["var_b"][e]
        put("db_mu", e, (E, N), vb * dm.sum(0), vb * np.abs(dm).sum(0), S + 4)
        put("db_var", e, (E, N), vb * vb * dv.sum(0), vb * vb * np.abs(dv).sum(0), S + 6)
    return out


# ---- routing -----------------------------------------------------------------------------

def route(mu_s, var_s, k):
    """The choice and the plan, token by token and expert by expert."""
    s = mu_s.astype(np.float64)
    T, E = s.shape
    expert = np.full((T, k), -1, np.int32)
    mu_g, var_g, jcb_g = (np.zeros((T, k)) for _ in range(3))
    for t in range(T):
        able = [e for e in range(E) if s[t, e] > -np.inf]
        able.sort(key=lambda e: (-s[t, e], e))
        able = able[:k]
        if not able:
            continue
        top = s[t, able[0]]
        w = np.array([1.0 if s[t, e] == top else np.exp(s[t, e] - top) for e in able])
        others = np.array([sum(w[:i]) + sum(w[i + 1:]) for i in range(len(w))])
        n = len(able)
        expert[t, :n] = able
        mu_g[t, :n] = w / w.sum()
        jcb_g[t, :n] = mu_g[t, :n] * others / w.sum()
        var_g[t, :n] = jcb_g[t, :n] ** 2 * var_s[t, able]
    offsets, token, slot = [0], [], np.full((T, k), -1, np.int32)
    for e in range(E):
        for t, j in zip(*np.nonzero(expert == e)):
            slot[t, j] = len(token)
            token.append(t)
        offsets.append(len(token))
    token += [-1] * (T * k - len(token))
    return dict(expert=expert, mu_g=mu_g, var_g=var_g, jcb_g=jcb_g, token=np.array(token, np.int32),
                offsets=np.array(offsets, np.int32), slot=slot)


def gate_bounds(mu_s, expert):
    """Relative bounds of a gate and of its slope. s - s_0 is rounded once, by at most U
    times its size, which expf turns into that relative error on top of its own (2 units in
    the last place, 4 U); the sum of k weights adds k roundings, the quotient one."""
    k = expert.shape[1]
    s = np.where(expert >= 0, np.take_along_axis(mu_s.astype(np.float64), np.maximum(expert, 0), 1), np.nan)
    with np.errstate(invalid="ignore"):
        gap = np.abs(s[:, :1] - s)
    gap = np.where(np.isfinite(gap), gap, 0.0).max(1, keepdims=True)
    g = (2 * gap + 8 + k + 2) * U
    return g, 2 * g + 2 * U


def combine_fwd(mu_g, var_g, mu_y, var_y, slot):
    g, vg, y, v = (a.astype(np.float64) for a in (mu_g, var_g, mu_y, var_y))
    T, k = slot.shape
    ok = (slot >= 0) & (slot < y.shape[0])
    at = np.where(ok, slot, 0)
    y, v = np.where(ok[..., None], y[at], 0.0), np.where(ok[..., None], v[at], 0.0)
    m = g[..., None] * y
    q = (g ** 2 + vg)[..., None] * v + vg[..., None] * y ** 2
    return dict(mu_z=(m.sum(1), (k + 2) * U * np.abs(m).sum(1)), var_z=(q.sum(1), (2 * k + 6) * U * q.sum(1)))


def combine_bwd(mu_g, jcb_g, mu_y, expert, slot, dmu, dvar, E):
    """Rows that nobody names stay NaN in the values."""
    g, jc, y, dm, dv = (a.astype(np.float64) for a in (mu_g, jcb_g, mu_y, dmu, dvar))
    T, k = slot.shape
    R, N = y.shape
    dy_mu, dy_var = np.full((R, N), np.nan), np.full((R, N), np.nan)
    ds = {x: np.zeros((T, E)) for x in ("mu", "var", "e_mu", "e_var")}
    for t in range(T):
        for j in range(k):
            r, e = slot[t, j], expert[t, j]
            if r < 0 or r >= R:
                continue
            dy_mu[r], dy_var[r] = g[t, j] * dm[t], g[t, j] ** 2 * dv[t]
            ds["mu"][t, e] += jc[t, j] * (y[r] * dm[t]).sum()
            ds["var"][t, e] += jc[t, j] ** 2 * (y[r] ** 2 * dv[t]).sum()
            ds["e_mu"][t, e] += (N + 4) * U * jc[t, j] * np.abs(y[r] * dm[t]).sum()
            ds["e_var"][t, e] += (N + 6) * U * jc[t, j] ** 2 * np.abs(y[r] ** 2 * dv[t]).sum()
    return dict(dy_mu=(dy_mu, 2 * U * np.abs(dy_mu)), dy_var=(dy_var, 3 * U * np.abs(dy_var)),
                ds_mu=(ds["mu"], ds["e_mu"]), ds_var=(ds["var"], ds["e_var"]))


def gather_bwd(dm, dv, slot, jcb=None, res=None):
    T, k = slot.shape
    ok = ((slot >= 0) & (slot < dm.shape[0]))[..., None]
    at = np.where(ok[..., 0], slot, 0)
    out = {}
    for name, x, i in (("mu", dm, 0), ("var", dv, 1)):
        rows = np.where(ok, x.astype(np.float64)[at], 0.0)
        r = np.zeros(rows[:, 0].shape) if res is None else res[i].astype(np.float64)
        j = 1.0 if jcb is None else jcb.astype(np.float64) ** (i + 1)
        size = (np.abs(rows).sum(1) + np.abs(r)) * np.abs(j)
        out[name] = ((rows.sum(1) + r) * j, (k + 4) * U * size)
    return out
