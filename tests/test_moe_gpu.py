"""Expert-grouped Linear layers, the router and the gated sum through the tensor-level calls
against their formulas in 64 bits, one by one and as the feed-forward block they make up."""
import numpy as np
import pytest

import moe_cases as C

pytestmark = pytest.mark.gpu

BWD = ("dz_mu", "dz_var", "dw_mu", "dw_var", "db_mu", "db_var")


def _dev(d):
    import torch
    return {k: None if v is None else torch.from_numpy(v).cuda() for k, v in d.items()}


def _host(t):
    return t.cpu().numpy()


@pytest.fixture(params=["by_size", "few_rows", "tiled"])
def kernel_choice(request):
    """Calls with few rows per expert go to kernels of their own; "few_rows" and "tiled" send
    every call to the ones or the others, so that the small shapes reach both."""
    from cutagi_amd import capi
    capi.tune("grouped.rows", {"by_size": -1, "few_rows": 1, "tiled": 0}[request.param])
    yield request.param
    capi.tune("grouped.rows", -1)


@pytest.fixture
def large_memory():
    """Gives the memory back to the device afterwards."""
    import torch
    yield
    torch.cuda.empty_cache()


# (rows of the experts, K, N, tokens or None, rows behind the last group)
GROUPS = [
    ([1], 1, 1, None, 0),
    ([3], 5, 7, None, 0),
    ([0, 1, 0], 16, 4, None, 0),
    ([2, 0, 5, 1], 33, 65, 3, 0),
    ([1, 1], 512, 256, 1, 0),
    ([7, 16, 17, 0, 3], 128, 96, None, 2),
    ([64, 63, 65, 1], 64, 128, 50, 0),
    ([130, 5, 0, 129], 96, 200, None, 9),
    ([40, 300, 1, 31], 260, 132, 100, 3),
    ([257, 128], 130, 66, None, 0),
    ([300], 515, 129, 64, 1),
    ([0, 0, 0], 32, 32, None, 4),
    ([1] * 40, 64, 64, 7, 0),
    ([9, 0, 12, 4] * 5, 72, 68, 30, 6),
    ([512, 600], 256, 256, None, 0),
    # more tiles than workgroups: every pass has workgroups that walk several
    ([130, 700, 0, 450], 4100, 72, 300, 5),
    ([130, 700, 0, 450], 72, 4100, None, 5),
    ([33, 90, 40], 1300, 1284, 100, 0),
    # the same with tiles of 64 rows
    ([50, 64, 0, 33] * 9, 40, 1284, 60, 0),
    ([50, 64, 0, 33] * 9, 1284, 40, None, 3),
    # long reductions of few tiles, taken in parts: of every pass, and parts of no rows
    ([700, 0, 300, 5], 523, 20, None, 3),
    ([40, 0, 200, 31], 2051, 37, 90, 0),
    ([150, 90], 70, 2050, None, 7),
    ([3000, 130], 36, 132, 77, 0),
    ([0, 1500, 0], 129, 6, 2, 100),
]
GUARD = 12345.0


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("sizes,K,N,tokens,tail", GROUPS)
def test_grouped_linear(kernel_choice, sizes, K, N, tokens, tail, bias):
    import torch
    import cutagi_amd.functional as F
    d = C.grouped_inputs(sizes, K, N, seed=K + N, tokens=tokens, tail=tail)
    t = _dev(d)
    R, total = t["dmu"].shape[0], sum(sizes)
    b = (t["mu_b"], t["var_b"]) if bias else (None, None)
    full = lambda *s: torch.full(s, GUARD, device="cuda")
    out = (full(R, N), full(R, N))
    F.grouped_linear_fwd(t["mu_w"], t["var_w"], *b, t["mu_a"], t["var_a"], t["offsets"], t["rows"], out)
    want = C.grouped_fwd(d, bias)
    for name, g in zip(("mu_z", "var_z"), out):
        C.check(_host(g)[:total], *want[name], name)
        assert np.all(_host(g)[total:] == GUARD), "rows behind the last group were written"
    for jcb in (True, False):
        E = len(sizes)
        out = [full(R, K), full(R, K), full(E, N, K), full(E, N, K), full(E, N), full(E, N)]
        got = F.grouped_linear_bwd(t["mu_w"], t["var_w"], b[1], t["mu_a"], t["jcb"] if jcb else None,
                                   t["dmu"], t["dvar"], t["offsets"], t["rows"], out=out)
        ref = C.grouped_bwd(d, jcb)
        for name, g in zip(BWD, got):
            if name[:2] == "db" and not bias:
                assert g is None
                continue
            g = _host(g)
            if name[:2] == "dz":
                assert np.all(g[total:] == GUARD), "rows behind the last group were written"
                g = g[:total]
            C.check(g, *ref[name], name)


@pytest.mark.parametrize("sizes,K,N,tokens", [([5, 0, 20], 96, 64, None), ([70, 130], 132, 260, 40),
                                              ([2, 1], 256, 128, 2), ([300, 0, 90], 600, 130, 70)])
def test_parts_and_the_same_bits_every_call(kernel_choice, sizes, K, N, tokens):
    import torch
    import cutagi_amd.functional as F
    t = _dev(C.grouped_inputs(sizes, K, N, seed=1, tokens=tokens))
    fwd = lambda: F.grouped_linear_fwd(t["mu_w"], t["var_w"], t["mu_b"], t["var_b"], t["mu_a"],
                                       t["var_a"], t["offsets"], t["rows"])
    bwd = lambda **kw: F.grouped_linear_bwd(t["mu_w"], t["var_w"], t["var_b"], t["mu_a"], t["jcb"],
                                            t["dmu"], t["dvar"], t["offsets"], t["rows"], **kw)
    z, g = fwd(), bwd()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(z + g, fwd() + bwd()))
    state, param = bwd(param_update=False), bwd(state_update=False)
    assert state[2:] == (None,) * 4 and param[:2] == (None,) * 2
    assert all(torch.equal(a, b) for a, b in zip(g, state[:2] + param[2:]))


@pytest.mark.parametrize("activation", ["relu", "mixture_relu"])
@pytest.mark.parametrize("sizes,K,N", [([3, 0, 2], 64, 40), ([90, 40], 72, 130), ([90, 0, 41], 777, 66)])
def test_fused_activation_is_the_activation_of_the_layer(kernel_choice, activation, sizes, K, N):
    import torch
    import cutagi_amd.functional as F
    t = _dev(C.grouped_inputs(sizes, K, N, seed=2, tokens=11))
    args = (t["mu_w"], t["var_w"], t["mu_b"], t["var_b"], t["mu_a"], t["var_a"], t["offsets"])
    mu, var = F.grouped_linear_fwd(*args, rows=t["rows"])
    want = (F.relu_fwd if activation == "relu" else F.mixture_relu_fwd)(mu, var)
    got = F.grouped_linear_fwd_act(*args, activation, rows=t["rows"])
    # the same sums go through the same device function: equal but for the contraction of its
    # multiplications and additions, a few roundings of terms no larger than mu^2 + var
    scale = (mu * mu + var + mu.abs() + 1).double()
    for name, g, w in zip(("mu", "var", "jcb"), got, want):
        C.check(_host(g), _host(w), 16 * C.U * _host(scale), name)


@pytest.mark.parametrize("sizes,K,N", [([5, 9], 64, 32), ([100, 31], 128, 132), ([140, 150], 260, 256),
                                       ([300, 270], 520, 518)])
def test_arrays_that_are_not_16_byte_aligned(kernel_choice, sizes, K, N):
    import torch
    import cutagi_amd.functional as F
    d = C.grouped_inputs(sizes, K, N, seed=4, tokens=30)

    def off(a):
        buf = torch.full((a.size + 8,), float("nan"), device="cuda")
        view = buf[1:1 + a.size].view(a.shape)
        view.copy_(torch.from_numpy(a))
        return view
    t = {k: off(v) if v.dtype == np.float32 else torch.from_numpy(v).cuda() for k, v in d.items()}
    got = F.grouped_linear_fwd(t["mu_w"], t["var_w"], t["mu_b"], t["var_b"], t["mu_a"], t["var_a"],
                               t["offsets"], t["rows"])
    for name, g in zip(("mu_z", "var_z"), got):
        C.check(_host(g), *C.grouped_fwd(d)[name], name)
    got = F.grouped_linear_bwd(t["mu_w"], t["var_w"], t["var_b"], t["mu_a"], t["jcb"], t["dmu"],
                               t["dvar"], t["offsets"], t["rows"])
    for name, g in zip(BWD, got):
        C.check(_host(g), *C.grouped_bwd(d)[name], name)


def test_indices_outside_the_arrays_read_nothing(kernel_choice):
    """Row indices that are no token stand for rows of zeros, offsets beyond the rows are
    moved to their end."""
    import torch
    import cutagi_amd.functional as F
    d = C.grouped_inputs([20, 30], 64, 48, seed=7, tokens=25)
    d["rows"][[0, 7, 33]] = [-1, 25, 2 ** 31 - 1]
    t = _dev(d)
    offsets = t["offsets"].clone()
    offsets[0], offsets[-1] = -5, 2 ** 30
    got = F.grouped_linear_fwd(t["mu_w"], t["var_w"], t["mu_b"], t["var_b"], t["mu_a"], t["var_a"],
                               offsets, t["rows"])
    for name, g in zip(("mu_z", "var_z"), got):
        C.check(_host(g), *C.grouped_fwd(d)[name], name)
    got = F.grouped_linear_bwd(t["mu_w"], t["var_w"], t["var_b"], t["mu_a"], t["jcb"], t["dmu"],
                               t["dvar"], offsets, t["rows"])
    for name, g in zip(BWD, got):
        C.check(_host(g), *C.grouped_bwd(d)[name], name)


@pytest.mark.parametrize("sizes,K,N,tail", [([5, 0, 9], 40, 36, 6), ([100, 31], 130, 64, 90), ([300, 0, 90], 600, 130, 20)])
def test_rows_behind_the_last_group_are_not_read(kernel_choice, sizes, K, N, tail):
    import torch
    import cutagi_amd.functional as F
    d = C.grouped_inputs(sizes, K, N, seed=3, tail=tail)
    t, total = _dev(d), sum(sizes)
    for name in ("mu_a", "var_a", "jcb", "dmu", "dvar"):
        t[name][total:] = float("nan")
    out = F.grouped_linear_fwd(t["mu_w"], t["var_w"], t["mu_b"], t["var_b"], t["mu_a"], t["var_a"], t["offsets"])
    want = {k: (v[0][:total], v[1][:total]) for k, v in C.grouped_fwd(d).items()}
    for name, g in zip(("mu_z", "var_z"), out):
        C.check(_host(g)[:total], *want[name], name)
    got = F.grouped_linear_bwd(t["mu_w"], t["var_w"], t["var_b"], t["mu_a"], t["jcb"], t["dmu"], t["dvar"],
                               t["offsets"])
    for name, g in zip(BWD, got):
        g = _host(g)
        C.check(g[:total] if name[:2] == "dz" else g, *C.grouped_bwd(d)[name], name)


def test_tokens_beyond_32_bit_offsets(kernel_choice, large_memory):
    """The last tokens of activations of more than 2^31 elements."""
    import torch
    import cutagi_amd.functional as F
    K, N, held, T = 16, 24, 50, (1 << 27) + 9
    d = C.grouped_inputs([150, 0, 40], K, N, seed=6, tokens=held)
    t = _dev(d)
    for name in ("mu_a", "var_a"):
        whole = torch.zeros(T, K, device="cuda")
        whole[T - held:] = t[name]
        t[name] = whole
    rows = t["rows"] + (T - held)
    got = F.grouped_linear_fwd(t["mu_w"], t["var_w"], t["mu_b"], t["var_b"], t["mu_a"], t["var_a"],
                               t["offsets"], rows)
    for name, g in zip(("mu_z", "var_z"), got):
        C.check(_host(g), *C.grouped_fwd(d)[name], name)
    got = F.grouped_linear_bwd(t["mu_w"], t["var_w"], t["var_b"], t["mu_a"], t["jcb"], t["dmu"],
                               t["dvar"], t["offsets"], rows)
    for name, g in zip(BWD, got):
        C.check(_host(g), *C.grouped_bwd(d)[name], name)


@pytest.mark.parametrize("sizes,K,N", [([300, 0, 90], 600, 130), ([700, 31], 523, 20)])
def test_two_graphs_replayed_side_by_side(sizes, K, N):
    """Calls that take their reductions in parts, recorded twice: each recording holds scratch
    memory of its own."""
    import torch
    import cutagi_amd.functional as F
    from cutagi_amd import capi
    assert capi.grouped_linear_scratch(K, N, len(sizes), sum(sizes)) > 0
    t = _dev(C.grouped_inputs(sizes, K, N, seed=8, tokens=200))

    def both():
        z = F.grouped_linear_fwd(t["mu_w"], t["var_w"], t["mu_b"], t["var_b"], t["mu_a"], t["var_a"],
                                 t["offsets"], t["rows"])
        return z + F.grouped_linear_bwd(t["mu_w"], t["var_w"], t["var_b"], t["mu_a"], t["jcb"], t["dmu"],
                                        t["dvar"], t["offsets"], t["rows"])
    both()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    held = []
    for g in graphs:
        with torch.cuda.graph(g):
            held.append(both())
    streams = [torch.cuda.Stream() for _ in graphs]
    for i in range(4):
        t["mu_a"].mul_(-1.1)
        want = both()
        torch.cuda.synchronize()
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for out in held:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), "replay %d" % i


def test_one_group_is_the_linear_layer(kernel_choice):
    """E = 1 against the ungrouped entry points (each is within its own bound of the exact
    result, so they are within twice that of one another)."""
    import cutagi_amd.functional as F
    d = C.grouped_inputs([96], 256, 128, seed=12)
    t = _dev(d)
    got = F.grouped_linear_fwd(t["mu_w"], t["var_w"], t["mu_b"], t["var_b"], t["mu_a"], t["var_a"],
                               t["offsets"])
    w = [t[k][0].contiguous() for k in ("mu_w", "var_w", "mu_b", "var_b")]
    for name, g, r in zip(("mu_z", "var_z"), got, F.linear_fwd(*w, t["mu_a"], t["var_a"])):
        C.check(_host(g), _host(r), 2 * C.grouped_fwd(d)[name][1], name)
    got = F.grouped_linear_bwd(t["mu_w"], t["var_w"], t["var_b"], t["mu_a"], t["jcb"], t["dmu"],
                               t["dvar"], t["offsets"])
    ref = F.linear_bwd(w[0], w[1], w[3], t["mu_a"], t["jcb"], t["dmu"], t["dvar"])
    for name, g, r in zip(BWD, got, ref):
        bound = 2 * C.grouped_bwd(d)[name][1]
        C.check(_host(g).reshape(_host(r).shape), _host(r), bound.reshape(_host(r).shape), name)


def test_innovations_against_differences(kernel_choice):
    """mu_z is linear in mu_a and in mu_w: <mu_z(a + v) - mu_z(a), delta_mu> = <v, delta_mu_z>
    without a Jacobian, and the same for the weights with delta_mu_w / var_w. Inputs in a few
    bits, so that the differences are exact."""
    import torch
    import cutagi_amd.functional as F
    rng = np.random.default_rng(3)
    few = lambda *s: torch.from_numpy(rng.integers(-4, 5, s).astype(np.float32)).cuda()
    sizes, K, N = [33, 0, 70], 40, 36
    E, R = 3, 103
    off = torch.tensor([0, 33, 33, 103], dtype=torch.int32, device="cuda")
    w, dw, a, da, dm = few(E, N, K), few(E, N, K), few(R, K), few(R, K), few(R, N)
    one, zero = torch.ones_like(w), torch.zeros_like(a)
    z = lambda w, a: F.grouped_linear_fwd(w, one, None, None, a, zero, off)[0].double()
    g = F.grouped_linear_bwd(w, one, None, a, None, dm, -dm.abs(), off)
    assert float(((z(w, a + da) - z(w, a)) * dm.double()).sum()) == float((g[0].double() * da.double()).sum())
    assert float(((z(w + dw, a) - z(w, a)) * dm.double()).sum()) == float((g[2].double() * dw.double()).sum())


# ---- router -------------------------------------------------------------------------------

ROUTES = [(1, 1, 1), (1, 8, 2), (33, 6, 3), (64, 40, 5), (3, 2, 2), (32, 16, 2), (5, 64, 64), (128, 6, 3), (129, 6, 3), (257, 65, 4),
          (1000, 3, 1), (300, 200, 8), (77, 1024, 5), (700, 1000, 33), (9000, 5, 2)]


def _check_route(mu_s, var_s, k):
    import torch
    import cutagi_amd.functional as F
    got = F.moe_route(torch.from_numpy(mu_s).cuda(), torch.from_numpy(var_s).cuda(), k)
    want = C.route(mu_s, var_s, k)
    for name in ("expert", "offsets", "token", "slot"):
        assert np.array_equal(_host(getattr(got, name)), want[name]), name
    g, s = C.gate_bounds(mu_s, want["expert"])
    # (values below the smallest normal number are rounded in steps of 2^-149)
    C.check(_host(got.mu_g), want["mu_g"], g * want["mu_g"] + 2.0 ** -126, "mu_g")
    C.check(_host(got.jcb_g), want["jcb_g"], s * want["jcb_g"] + 2.0 ** -126, "jcb_g")
    C.check(_host(got.var_g), want["var_g"], (2 * s + 2 * C.U) * want["var_g"] + 2.0 ** -126, "var_g")
    return got


@pytest.mark.parametrize("T,E,k", ROUTES)
def test_route(T, E, k):
    rng = np.random.default_rng(T + E)
    mu = (2 * rng.standard_normal((T, E))).astype(np.float32)
    _check_route(mu, rng.uniform(0.01, 0.5, (T, E)).astype(np.float32), k)


@pytest.mark.parametrize("T,E,k", [(40, 7, 3), (500, 33, 4)])
def test_route_ties_and_masked_scores(T, E, k):
    """Scores in few steps (ties everywhere, zeros of both signs), -inf and NaN in masked
    places, tokens without any expert left, and infinite scores."""
    rng = np.random.default_rng(T)
    mu = rng.integers(-2, 3, (T, E)).astype(np.float32)
    mu[rng.random((T, E)) < 0.1] *= -0.0
    mu[rng.random((T, E)) < 0.3] = -np.inf
    mu[rng.random((T, E)) < 0.1] = np.nan
    mu[3] = -np.inf
    mu[4] = np.nan
    mu[5, 2:4] = np.inf
    mu[6] = np.finfo(np.float32).min      # a mask of the type's lowest value: they tie
    mu[7, :] = -np.inf
    mu[7, E - 1] = np.finfo(np.float32).min
    got = _check_route(mu, rng.uniform(0.01, 0.5, (T, E)).astype(np.float32), k)
    assert np.all(_host(got.expert)[3:5] == -1) and np.all(_host(got.mu_g)[3:5] == 0)
    assert _host(got.expert)[7, 0] == E - 1 and _host(got.mu_g)[7, 0] == 1


def test_plan_of_more_tokens_than_31_bits_of_threads(large_memory):
    """Eight threads per token look for places behind the last row: past 2^28 tokens their
    numbers leave 31 bits."""
    import torch
    import cutagi_amd.functional as F
    T = (1 << 28) + 33
    mu = torch.zeros(T, 1, device="cuda")
    mu[::1000] = -float("inf")
    mu[-5:] = -float("inf")
    live = (mu[:, 0] == 0).nonzero()[:, 0].int()
    n = live.numel()
    r = F.moe_route(mu, torch.full_like(mu, 0.1), 1)
    assert r.offsets.tolist() == [0, n]
    assert torch.equal(r.token[:n], live) and bool((r.token[n:] == -1).all())
    slot = torch.full((T,), -1, dtype=torch.int32, device="cuda")
    slot[live.long()] = torch.arange(n, dtype=torch.int32, device="cuda")
    assert torch.equal(r.slot[:, 0], slot)
    assert torch.equal(r.expert[:, 0], torch.where(slot >= 0, 0, -1).int())
    assert torch.equal(r.mu_g, (r.expert >= 0).float())



def test_slope_of_the_gates_against_differences():
    import torch
    import cutagi_amd.functional as F
    rng = np.random.default_rng(0)
    mu = torch.from_numpy(rng.standard_normal((64, 8)).astype(np.float32)).cuda()
    var = torch.full_like(mu, 0.1)
    r = F.moe_route(mu, var, 3)
    h = 2.0 ** -6
    for j in range(3):
        step = torch.zeros_like(mu).scatter_(1, r.expert[:, j:j + 1].long(), h)
        up, down = F.moe_route(mu + step, var, 8), F.moe_route(mu - step, var, 8)
        # all eight experts chosen: compare the softmax over the three that r chose
        pick = lambda q: torch.zeros_like(mu).scatter_(1, q.expert.long(), q.mu_g)
        gate = lambda p: p.gather(1, r.expert.long()) / p.gather(1, r.expert.long()).sum(1, keepdim=True)
        slope = ((gate(pick(up)) - gate(pick(down))) / (2 * h))[:, j].double()
        # the central difference of a sigmoid is off by h^2/6 times its third derivative (below
        # 1/8) and by the rounding of the gates over 2 h
        assert float((slope - r.jcb_g[:, j].double()).abs().max()) <= h * h / 48 + 64 * C.U / (2 * h)


# ---- gated sum ------------------------------------------------------------------------------

def _gated(T, E, k, N, seed, masked=0.2):
    rng = np.random.default_rng(seed)
    mu = rng.standard_normal((T, E)).astype(np.float32)
    mu[rng.random((T, E)) < masked] = -np.inf
    r = C.route(mu, rng.uniform(0.01, 0.5, (T, E)).astype(np.float32), k)
    d = {n: r[n].astype(np.float32) for n in ("mu_g", "var_g", "jcb_g")}
    f = np.float32
    d.update(expert=r["expert"], slot=r["slot"], mu_y=rng.standard_normal((T * k, N)).astype(f),
             var_y=rng.uniform(0.01, 0.5, (T * k, N)).astype(f),
             dmu=(0.1 * rng.standard_normal((T, N))).astype(f), dvar=(-rng.uniform(0, 1e-2, (T, N))).astype(f))
    return d


@pytest.mark.parametrize("T,E,k,N", [(1, 2, 2, 1), (1, 8, 2, 4096), (7, 5, 3, 33), (40, 4, 1, 64), (33, 16, 4, 1028),
                                     (20, 6, 2, 1025), (9, 70, 5, 2049), (300, 3, 2, 12)])
def test_gated_sum(T, E, k, N):
    import torch
    import cutagi_amd.functional as F
    d = _gated(T, E, k, N, seed=T + N)
    t = _dev(d)
    got = F.moe_combine_fwd(t["mu_g"], t["var_g"], t["mu_y"], t["var_y"], t["slot"])
    for name, g in zip(("mu_z", "var_z"), got):
        C.check(_host(g), *C.combine_fwd(d["mu_g"], d["var_g"], d["mu_y"], d["var_y"], d["slot"])[name], name)
    out = [torch.full((T * k, N), float("nan"), device="cuda") for _ in range(2)]
    got = F.moe_combine_bwd(t["mu_g"], t["jcb_g"], t["mu_y"], t["expert"], t["slot"], t["dmu"], t["dvar"], E, out=out)
    want = C.combine_bwd(d["mu_g"], d["jcb_g"], d["mu_y"], d["expert"], d["slot"], d["dmu"], d["dvar"], E)
    for name, g in zip(("dy_mu", "dy_var", "ds_mu", "ds_var"), got):
        value, bound = want[name]
        g, live = _host(g), ~np.isnan(value)
        assert np.all(np.isnan(g[~live])), name + ": rows that nobody names were written"
        C.check(g[live], value[live], bound[live], name)
    for jcb in (None, "dmu"):
        for res in (None, ("dmu", "dvar")):
            rows = (t["mu_y"], t["var_y"])
            g = F.moe_gather_bwd(*rows, t["slot"], t[jcb] if jcb else None, *((t[r] for r in res) if res else ()))
            w = C.gather_bwd(d["mu_y"], d["var_y"], d["slot"], d[jcb] if jcb else None,
                             [d[r] for r in res] if res else None)
            C.check(_host(g[0]), *w["mu"], "gathered mu")
            C.check(_host(g[1]), *w["var"], "gathered var")


def test_gated_sum_of_rows_beyond_32_bit_offsets(large_memory):
    """The last rows of expert outputs of more than 2^31 elements."""
    import torch
    import cutagi_amd.functional as F
    T, E, k, N = 6, 4, 2, 4100
    d = _gated(T, E, k, N, seed=5)
    t, held = _dev(d), T * k
    R = (1 << 19) + held
    for name in ("mu_y", "var_y"):
        whole = torch.zeros(R, N, device="cuda")
        whole[R - held:] = t[name]
        t[name] = whole
    slot = torch.where(t["slot"] >= 0, t["slot"] + (R - held), t["slot"])
    got = F.moe_combine_fwd(t["mu_g"], t["var_g"], t["mu_y"], t["var_y"], slot)
    for name, g in zip(("mu_z", "var_z"), got):
        C.check(_host(g), *C.combine_fwd(d["mu_g"], d["var_g"], d["mu_y"], d["var_y"], d["slot"])[name], name)
    g = F.moe_gather_bwd(t["mu_y"], t["var_y"], slot)
    w = C.gather_bwd(d["mu_y"], d["var_y"], d["slot"])
    C.check(_host(g[0]), *w["mu"], "gathered mu")
    C.check(_host(g[1]), *w["var"], "gathered var")
    got = F.moe_combine_bwd(t["mu_g"], t["jcb_g"], t["mu_y"], t["expert"], slot, t["dmu"], t["dvar"], E)
    want = C.combine_bwd(d["mu_g"], d["jcb_g"], d["mu_y"], d["expert"], d["slot"], d["dmu"], d["dvar"], E)
    for name, g in zip(("dy_mu", "dy_var", "ds_mu", "ds_var"), got):
        value, bound = want[name]
        g, live = _host(g[R - held:] if name[:2] == "dy" else g), ~np.isnan(value)
        C.check(g[live], value[live], bound[live], name)


# ---- as they are used ------------------------------------------------------------------------

def _block_inputs(T, n, H, E, seed):
    rng = np.random.default_rng(seed)
    f = np.float32
    norm = C.norm_inputs(T, n, seed)
    d = {"n_" + k: v for k, v in norm.items()}
    d.update(r_mu_w=rng.normal(0, n ** -0.5, (E, n)).astype(f), r_var_w=(rng.uniform(.5, 1.5, (E, n)) / n).astype(f))
    for name, N, K in (("u", H, n), ("d", n, H)):
        d[name + "_mu_w"] = rng.normal(0, K ** -0.5, (E, N, K)).astype(f)
        d[name + "_var_w"] = (rng.uniform(.5, 1.5, (E, N, K)) / K).astype(f)
        d[name + "_mu_b"] = rng.normal(0, .2, (E, N)).astype(f)
        d[name + "_var_b"] = (rng.uniform(.5, 1.5, (E, N)) / K).astype(f)
    return d


def _block(t, k, E):
    """Pre-norm feed-forward block with experts: every output of its forward and backward."""
    import cutagi_amd.functional as F
    mu_z, var_z, m, v = F.layernorm_fwd(t["n_mu_w"], t["n_var_w"], t["n_mu_b"], t["n_var_b"], t["n_mu_a"], t["n_var_a"])
    mu_s, var_s = F.linear_fwd(t["r_mu_w"], t["r_var_w"], None, None, mu_z, var_z)
    r = F.moe_route(mu_s, var_s, k)
    up = [t["u_" + x] for x in ("mu_w", "var_w", "mu_b", "var_b")]
    down = [t["d_" + x] for x in ("mu_w", "var_w", "mu_b", "var_b")]
    mu_h, var_h, jcb_h = F.grouped_linear_fwd_act(*up, mu_z, var_z, r.offsets, "relu", rows=r.token)
    mu_y, var_y = F.grouped_linear_fwd(*down, mu_h, var_h, r.offsets)
    out = F.moe_combine_fwd(r.mu_g, r.var_g, mu_y, var_y, r.slot)
    dmu, dvar = t["n_dmu"], t["n_dvar"]
    dy_mu, dy_var, ds_mu, ds_var = F.moe_combine_bwd(r.mu_g, r.jcb_g, mu_y, r.expert, r.slot, dmu, dvar, E)
    gd = F.grouped_linear_bwd(down[0], down[1], down[3], mu_h, jcb_h, dy_mu, dy_var, r.offsets)
    gu = F.grouped_linear_bwd(up[0], up[1], up[3], mu_z, None, gd[0], gd[1], r.offsets, rows=r.token)
    import torch
    gr = F.linear_bwd(t["r_mu_w"], t["r_var_w"], None, mu_z, torch.ones_like(mu_z), ds_mu, ds_var)
    dz = F.moe_gather_bwd(gu[0], gu[1], r.slot, None, gr[0], gr[1])
    gn = F.layernorm_bwd(t["n_mu_w"], t["n_var_w"], t["n_var_b"], t["n_mu_a"], t["n_jcb"], m, v, *dz)
    return r, list(out) + list(gd[2:]) + list(gu[2:]) + list(gr[2:4]) + list(gn)


def _block_64(d, r, k, E):
    """The same block in 64 bits, with the experts that the fp32 scores chose."""
    d = {n: v.astype(np.float64) for n, v in d.items()}
    a, q = d["n_mu_a"], d["n_var_a"]
    n = a.shape[1]
    m = a.mean(1, keepdims=True)
    inv = 1 / np.sqrt((((a - m) ** 2).sum(1, keepdims=True) + q.sum(1, keepdims=True)) / (n - 1) + 1e-5)
    x = inv * (a - m)
    z = x * d["n_mu_w"] + d["n_mu_b"]
    vz = inv ** 2 * q * (d["n_mu_w"] ** 2 + d["n_var_w"]) + d["n_var_w"] * x ** 2 + d["n_var_b"]
    lin = lambda w, v, mb, vb, i, j: (i @ w.T + mb, (j + i ** 2) @ v.T + j @ (w ** 2).T + vb)
    s, vs = lin(d["r_mu_w"], d["r_var_w"], 0, 0, z, vz)
    T = a.shape[0]
    mu, var = np.zeros((T, n)), np.zeros((T, n))
    dz, dvz = np.zeros((T, n)), np.zeros((T, n))
    ds, dvs = np.zeros((T, E)), np.zeros((T, E))
    g = {x: np.zeros_like(d[x]) for x in d if x[:2] in ("u_", "d_")}
    dm, dv = d["n_dmu"], d["n_dvar"]
    for t in range(T):
        es = r["expert"][t][r["expert"][t] >= 0]
        w = np.exp(s[t, es] - s[t, es].max())
        w /= w.sum()
        for e, gate in zip(es, w):
            slope = gate * (1 - gate)
            vg = slope ** 2 * vs[t, e]
            h, vh = lin(d["u_mu_w"][e], d["u_var_w"][e], d["u_mu_b"][e], d["u_var_b"][e], z[t:t + 1], vz[t:t + 1])
            j = (h > 0) * 1.0
            h, vh = h * j, vh * j
            y, vy = lin(d["d_mu_w"][e], d["d_var_w"][e], d["d_mu_b"][e], d["d_var_b"][e], h, vh)
            mu[t] += (gate * y)[0]
            var[t] += ((gate ** 2 + vg) * vy + vg * y ** 2)[0]
            dy, dvy = gate * dm[t:t + 1], gate ** 2 * dv[t:t + 1]
            ds[t, e], dvs[t, e] = slope * (y * dm[t]).sum(), slope ** 2 * (y ** 2 * dv[t]).sum()
            dh, dvh = (dy @ d["d_mu_w"][e]) * j, (dvy @ d["d_mu_w"][e] ** 2) * j
            for p, D, V, X in (("d_", dy, dvy, h), ("u_", dh, dvh, z[t:t + 1])):
                g[p + "mu_w"][e] += D.T @ X
                g[p + "var_w"][e] += V.T @ X ** 2
                g[p + "mu_b"][e] += D[0]
                g[p + "var_b"][e] += V[0]
            dz[t] += (dh @ d["u_mu_w"][e])[0]
            dvz[t] += (dvh @ d["u_mu_w"][e] ** 2)[0]
    dz, dvz = dz + ds @ d["r_mu_w"], dvz + dvs @ d["r_mu_w"] ** 2
    out = [mu, var]
    for p in ("d_", "u_"):
        out += [d[p + "var_w"] * g[p + "mu_w"], d[p + "var_w"] ** 2 * g[p + "var_w"],
                d[p + "var_b"] * g[p + "mu_b"], d[p + "var_b"] ** 2 * g[p + "var_b"]]
    out += [d["r_var_w"] * (ds.T @ z), d["r_var_w"] ** 2 * (dvs.T @ z ** 2)]
    t = inv * d["n_mu_w"] * d["n_jcb"]
    out += [t * dz, t ** 2 * dvz, d["n_var_w"] * (x * dz).sum(0), d["n_var_w"] ** 2 * (x ** 2 * dvz).sum(0),
            d["n_var_b"] * dz.sum(0), d["n_var_b"] ** 2 * dvz.sum(0)]
    return out


@pytest.mark.parametrize("T,n,H,E,k", [(1, 64, 96, 4, 2), (37, 48, 130, 5, 2), (200, 68, 40, 6, 3)])
def test_block(T, n, H, E, k):
    """All of the block against 64 bits. Norm-wise: every output is a chain of at most six
    sums of at most max(n, H, T E) terms; 6 (S + 16) U of the result's norm times 8 for the
    cancellation between its terms (inputs with random signs: a sum is about its terms'
    root of squares, sqrt(S) below their magnitudes' sum, S <= 1200 here)."""
    d = _block_inputs(T, n, H, E, seed=T)
    r, got = _block(_dev(d), k, E)
    choice = {x: _host(getattr(r, x)) for x in ("expert", "slot")}
    want = _block_64(d, choice, k, E)
    assert len(got) == len(want)
    S = max(n, H, T)
    for i, (g, w) in enumerate(zip(got, want)):
        g = _host(g).astype(np.float64).reshape(w.shape)
        assert np.all(np.isfinite(g))
        assert np.linalg.norm(g - w) <= 6 * (S + 16) * C.U * 8 * np.linalg.norm(w), "output %d" % i


def test_block_replayed_from_a_graph_and_on_another_stream():
    import torch
    d = _block_inputs(150, 64, 96, 6, seed=1)
    t = _dev(d)
    _block(t, 2, 6)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, held = _block(t, 2, 6)
    side = torch.cuda.Stream()
    for i in range(4):
        t["n_mu_a"].mul_(-1.1).add_(0.05)
        _, want = _block(t, 2, 6)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):       # at the same time, on a stream of its own
            _, other = _block(t, 2, 6)
        torch.cuda.synchronize()
        for j, (a, b, c) in enumerate(zip(held, want, other)):
            assert torch.equal(a, b), "replay %d, output %d" % (i, j)
            assert torch.equal(c, b), "side stream %d, output %d" % (i, j)
