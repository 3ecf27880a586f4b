"""Expert-grouped Linear layers on sums of a single term (see single_term_cases): every product of
every pass is as exact as six products of bf16 pieces make it, at any place of a long reduction
and whichever kernels take the call."""
import numpy as np
import pytest

import moe_cases as C
import single_term_cases as S

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["by_size", "few_rows", "tiled"])
def kernel_choice(request):
    from cutagi_amd import capi
    capi.tune("grouped.rows", {"by_size": -1, "few_rows": 1, "tiled": 0}[request.param])
    yield request.param
    capi.tune("grouped.rows", -1)


@pytest.mark.parametrize("sizes,K,N,tokens", [
    ([130, 5, 0, 129], 96, 200, None), ([40, 0, 200, 31], 2051, 37, 90), ([300], 515, 129, 64),
    ([700, 0, 300, 5], 523, 20, None), ([50, 64, 0, 33] * 6, 1284, 40, 60), ([150, 90], 70, 2050, None),
    ([3000, 130], 36, 132, 77), ([2, 0, 5, 1], 33, 65, 3), ([1], 4096, 256, None)])
def test_single_terms(kernel_choice, sizes, K, N, tokens):
    import torch
    import cutagi_amd.functional as F
    d = S.inputs(sizes, K, N, seed=K + N, tokens=tokens)
    t = {k: torch.from_numpy(v).cuda() for k, v in d.items() if v is not None}
    rows = t.get("rows")
    host = lambda a: a.cpu().numpy()
    fwd = S.forward(d)
    nothing = torch.zeros_like(t["mean"])
    mu, var = F.grouped_linear_fwd(t["mu_w"], t["var_w"], None, None, t["mean"], nothing, t["offsets"], rows)
    C.check(host(mu), *fwd["mu_z"], "mu_z")
    C.check(host(var), *fwd["var_z"], "var_z of the mean")
    mu, var = F.grouped_linear_fwd(t["mu_w"], torch.zeros_like(t["var_w"]), None, None, nothing, t["var"],
                                   t["offsets"], rows)
    assert float(mu.abs().max()) == 0
    C.check(host(var), *fwd["var_only"], "var_z of the variance")
    back = lambda m, v, **kw: F.grouped_linear_bwd(t["mu_w"], t["var_w"], None, t["mu_a"], None, t[m], t[v],
                                                   t["offsets"], rows, **kw)
    for name, got in zip(("dz_mu", "dz_var"), back("row_mu", "row_var", param_update=False)):
        C.check(host(got), *S.state_backward(d)[name], name)
    for name, got in zip(("dw_mu", "dw_var"), back("column_mu", "column_var", state_update=False)[2:4]):
        C.check(host(got), *S.weight_backward(d)[name], name)
