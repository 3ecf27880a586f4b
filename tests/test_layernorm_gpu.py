"""The layer norm through the tensor-level calls against its formulas in 64 bits."""
import numpy as np
import pytest

import moe_cases as C

pytestmark = pytest.mark.gpu

EPS = 1e-5
# (rows, features): one row, two features, odd sizes, every row width the kernels hold in
# registers and one beyond, with and without whole 16-byte groups
SHAPES = [(1, 2), (3, 3), (5, 13), (2, 64), (129, 65), (1, 1024), (67, 1000), (33, 1023), (4, 2048),
          (3, 4095), (2, 4096), (3, 4100), (2, 8191), (2, 8192), (2, 8196), (3, 9001), (1000, 7),
          (4099, 24), (2051, 260), (9001, 4), (70001, 2), (5000, 1001)]


def _dev(d):
    import torch
    return {k: torch.from_numpy(v).cuda() for k, v in d.items()}


def _host(t):
    return t.cpu().numpy()


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("B,n", SHAPES)
def test_forward_and_backward(B, n, bias):
    import cutagi_amd.functional as F
    d = C.norm_inputs(B, n, seed=B + n)
    t = _dev(d)
    b = (t["mu_b"], t["var_b"]) if bias else (None, None)
    got = F.layernorm_fwd(t["mu_w"], t["var_w"], *b, t["mu_a"], t["var_a"], EPS)
    want = C.norm_fwd(d, EPS, bias)
    for name, g in zip(("mu_z", "var_z", "mu_s", "var_s"), got):
        C.check(_host(g), *want[name], name)
    for jcb in (True, False):
        grads = F.layernorm_bwd(t["mu_w"], t["var_w"], b[1], t["mu_a"], t["jcb"] if jcb else None,
                                got[2], got[3], t["dmu"], t["dvar"], EPS)
        ref = C.norm_bwd(d, _host(got[2]), _host(got[3]), EPS, jcb)
        for name, g in zip(("dz_mu", "dz_var", "dw_mu", "dw_var", "db_mu", "db_var"), grads):
            if name[:2] == "db" and not bias:
                assert g is None
            else:
                C.check(_host(g), *ref[name], name)


def test_parts_of_the_backward_pass_and_the_same_bits_every_call():
    import torch
    import cutagi_amd.functional as F
    d = C.norm_inputs(777, 520, seed=3)
    t = _dev(d)
    _, _, m, v = F.layernorm_fwd(t["mu_w"], t["var_w"], None, None, t["mu_a"], t["var_a"], EPS)
    call = lambda **kw: F.layernorm_bwd(t["mu_w"], t["var_w"], t["var_b"], t["mu_a"], t["jcb"], m, v,
                                        t["dmu"], t["dvar"], EPS, **kw)
    full = call()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(full, call()))
    state, param = call(param_update=False), call(state_update=False)
    assert state[2:] == (None,) * 4 and param[:2] == (None,) * 2
    assert all(torch.equal(a, b) for a, b in zip(full[:2], state[:2]))
    assert all(torch.equal(a, b) for a, b in zip(full[2:], param[2:]))
    assert call(state_update=False, param_update=False) == (None,) * 6


@pytest.mark.parametrize("B,n", [(3, 64), (2, 1024), (5, 4096), (2, 8200)])
def test_arrays_that_are_not_16_byte_aligned(B, n):
    """Whole 16-byte groups per row, but every array starts 4 bytes behind a boundary."""
    import torch
    import cutagi_amd.functional as F
    d = C.norm_inputs(B, n, seed=9)

    def off(a):
        buf = torch.full((a.size + 8,), float("nan"), device="cuda")
        view = buf[1:1 + a.size].view(a.shape)
        view.copy_(torch.from_numpy(a))
        return view
    t = {k: off(v) for k, v in d.items()}
    got = F.layernorm_fwd(t["mu_w"], t["var_w"], t["mu_b"], t["var_b"], t["mu_a"], t["var_a"], EPS)
    for name, g in zip(("mu_z", "var_z", "mu_s", "var_s"), got):
        C.check(_host(g), *C.norm_fwd(d, EPS)[name], name)
    m, v = off(_host(got[2])), off(_host(got[3]))
    grads = F.layernorm_bwd(t["mu_w"], t["var_w"], t["var_b"], t["mu_a"], t["jcb"], m, v, t["dmu"],
                            t["dvar"], EPS)
    ref = C.norm_bwd(d, _host(m), _host(v), EPS)
    for name, g in zip(("dz_mu", "dz_var", "dw_mu", "dw_var", "db_mu", "db_var"), grads):
        C.check(_host(g), *ref[name], name)


def test_constant_rows_and_a_large_mean():
    """Rows whose features are all alike: no deviation, the variances alone; and rows whose
    mean is far larger than their spread, where sums of squares would cancel."""
    import cutagi_amd.functional as F
    d = C.norm_inputs(4, 300, seed=5)
    d["mu_a"][0] = 3.0
    d["mu_a"][1] = 0.0
    d["var_a"][1] = 0.0           # variance zero: only eps is left under the root
    d["mu_a"][2:] += 4096.0
    t = _dev(d)
    got = F.layernorm_fwd(t["mu_w"], t["var_w"], t["mu_b"], t["var_b"], t["mu_a"], t["var_a"], EPS)
    for name, g in zip(("mu_z", "var_z", "mu_s", "var_s"), got):
        C.check(_host(g), *C.norm_fwd(d, EPS)[name], name)


def test_weight_innovation_against_differences():
    """mu_z is linear in mu_w: sum_b (mu_z(mu_w + 1) - mu_z(mu_w)) delta_mu, feature by
    feature, is the mean innovation over var_w."""
    import torch
    import cutagi_amd.functional as F
    d = C.norm_inputs(50, 96, seed=6)
    t = _dev(d)
    at = lambda w: F.layernorm_fwd(w, t["var_w"], None, None, t["mu_a"], t["var_a"], EPS)
    zero = torch.zeros_like(t["mu_w"])
    low, high = at(zero), at(torch.ones_like(zero))
    diff = ((high[0] - low[0]).double() * t["dmu"].double()).sum(0)
    grad = F.layernorm_bwd(t["mu_w"], t["var_w"], None, t["mu_a"], None, low[2], low[3], t["dmu"],
                           t["dvar"], EPS)[2]
    # both sides carry the rounding of x (4 U) and of the sum of 50 products
    size = ((high[0] - low[0]).double() * t["dmu"].double()).abs().sum(0) * t["var_w"].double()
    C.check(_host(grad), _host(diff * t["var_w"].double()), (50 + 20) * C.U * _host(size), "dw_mu")


def test_replays_of_a_graph():
    import torch
    import cutagi_amd.functional as F
    d = C.norm_inputs(640, 512, seed=8)
    t = _dev(d)

    def step():
        z = F.layernorm_fwd(t["mu_w"], t["var_w"], t["mu_b"], t["var_b"], t["mu_a"], t["var_a"], EPS)
        return z + F.layernorm_bwd(t["mu_w"], t["var_w"], t["var_b"], t["mu_a"], t["jcb"], z[2], z[3],
                                   t["dmu"], t["dvar"], EPS)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        t["mu_a"].mul_(1.5).add_(0.1)
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), "replay %d" % i


@pytest.fixture
def large_memory():
    """Gives the memory back to the device afterwards."""
    import torch
    yield
    torch.cuda.empty_cache()


def test_more_than_32_bit_offsets(large_memory):
    """The last rows of 2^31 elements and more: each row as in a call of its own, the parameter
    innovations those of the only rows that have any (five of them)."""
    import torch
    import cutagi_amd.functional as F
    n, few = 4100, 5
    B = (1 << 19) + few
    d = C.norm_inputs(few, n, seed=10)
    t = _dev(d)
    whole = {}
    for name in ("mu_a", "var_a", "dmu", "dvar"):
        whole[name] = torch.zeros(B, n, device="cuda")
        whole[name][B - few:] = t[name]
    args = (t["mu_w"], t["var_w"], t["mu_b"], t["var_b"])
    want = F.layernorm_fwd(*args, t["mu_a"], t["var_a"], EPS)
    got = F.layernorm_fwd(*args, whole["mu_a"], whole["var_a"], EPS)
    for g, w in zip(got, want):
        assert torch.equal(g[B - few:], w)
    grads = F.layernorm_bwd(t["mu_w"], t["var_w"], t["var_b"], whole["mu_a"], None, got[2], got[3], whole["dmu"],
                            whole["dvar"], EPS)
    ref = C.norm_bwd(d, _host(want[2]), _host(want[3]), EPS, False)
    for name, g in zip(("dz_mu", "dz_var", "dw_mu", "dw_var", "db_mu", "db_var"), grads):
        C.check(_host(g[B - few:] if name[:2] == "dz" else g), *ref[name], name)
