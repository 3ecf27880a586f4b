"""LayerNorm and MixtureOfExperts as layers of a Sequential: the same bits as the tensor-level
calls they are made of (which have their own tests against 64 bits), through forward,
backward, parameter step, replayed graphs, blocks and checkpoints."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

N_IN, HIDDEN, N_OUT, EXPERTS, TOP_K = 24, 40, 12, 5, 2


def _net(cutagi, activation="relu", bias=True, seed=0, first=True):
    cutagi.manual_seed(seed)
    layers = [cutagi.Linear(16, N_IN), cutagi.MixtureReLU()] if first else []
    layers += [cutagi.LayerNorm([N_IN], 1e-5, bias),
               cutagi.MixtureOfExperts(N_IN, HIDDEN, N_OUT, EXPERTS, TOP_K, activation, bias)]
    net = cutagi.Sequential(layers)
    net.to_device("cuda")
    return net


def _params(net, name):
    import torch
    return [torch.tensor(x, dtype=torch.float32, device="cuda") if len(x) else None
            for x in net.state_dict()[name]]


def _split(p, bias):
    """(mu_w, var_w, mu_b, var_b) of the router, the first and the second expert layers."""
    E, K, H, N = EXPERTS, N_IN, HIDDEN, N_OUT
    ends = [0, E * K, E * K + E * H * K, E * K + E * H * K + E * N * H]
    bends = [0, E, E + E * H, E + E * H + E * N]
    shapes = [(E, K), (E, H, K), (E, N, H)]
    bshapes = [(E,), (E, H), (E, N)]
    out = []
    for i in range(3):
        w = [x[ends[i]:ends[i + 1]].reshape(shapes[i]) for x in p[:2]]
        b = [x[bends[i]:bends[i + 1]].reshape(bshapes[i]) if bias else None for x in p[2:]]
        out.append([t.clone() if t is not None else None for t in w + b])
    return out


@pytest.mark.parametrize("activation", ["relu", "mixture_relu"])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("batch", [1, 7, 300])
def test_layers_are_their_calls(batch, bias, activation):
    import torch
    import cutagi_amd.functional as F
    from cutagi_amd import capi, cutagi
    rng = np.random.default_rng(batch)
    f = np.float32
    net = _net(cutagi, activation, bias, first=False)
    net.input_state_update = True
    x, v = rng.standard_normal((batch, N_IN)).astype(f), rng.uniform(0.01, 0.2, (batch, N_IN)).astype(f)
    dmu, dvar = (0.1 * rng.standard_normal((batch, N_OUT))).astype(f), (-rng.uniform(0, 0.01, (batch, N_OUT))).astype(f)
    names = ("LayerNormCuda.0", "MixtureOfExpertsCuda.1")
    norm, moe = (_params(net, n) for n in names)
    net.forward(x, v)
    got = net.get_outputs()
    choices = np.array(net.layers[1].get_expert_choices()).reshape(batch, TOP_K)
    pad = np.zeros(net.input_delta_z_buffer.size - dmu.size, f)      # the buffer's whole length
    net.set_delta_z(np.concatenate([dmu.ravel(), pad]), np.concatenate([dvar.ravel(), pad]))
    net.backward()
    net.delta_z_to_host()
    back = [net.output_delta_z_buffer.delta_mu, net.output_delta_z_buffer.delta_var]
    net.step()

    t = lambda a: torch.from_numpy(a).cuda()
    z, vz, m, s = F.layernorm_fwd(*norm, t(x), t(v), 1e-5)
    router, up, down = _split(moe, bias)
    scores = F.linear_fwd(*router, z, vz)
    r = F.moe_route(*scores, TOP_K)
    h, vh, jh = F.grouped_linear_fwd_act(*up, z, vz, r.offsets, activation, rows=r.token)
    y, vy = F.grouped_linear_fwd(*down, h, vh, r.offsets)
    out = F.moe_combine_fwd(r.mu_g, r.var_g, y, vy, r.slot)
    for g, w in zip(got, out):
        assert np.array_equal(np.asarray(g).ravel(), w.cpu().numpy().ravel())
    assert np.array_equal(choices, r.expert.cpu().numpy())

    dy, dvy, ds, dvs = F.moe_combine_bwd(r.mu_g, r.jcb_g, y, r.expert, r.slot, t(dmu), t(dvar), EXPERTS)
    gd = F.grouped_linear_bwd(down[0], down[1], down[3], h, jh, dy, dvy, r.offsets)
    gu = F.grouped_linear_bwd(up[0], up[1], up[3], z, None, gd[0], gd[1], r.offsets, rows=r.token)
    gr = F.linear_bwd(router[0], router[1], router[3], z, torch.ones_like(z), ds, dvs)
    dz = F.moe_gather_bwd(gu[0], gu[1], r.slot, None, gr[0], gr[1])
    gn = F.layernorm_bwd(norm[0], norm[1], norm[3], t(x), None, m, s, *dz, 1e-5)
    for g, w in zip(back, gn[:2]):
        assert np.array_equal(np.asarray(g)[:batch * N_IN], w.cpu().numpy().ravel())

    # the step: every parameter through the same capped update
    cap = capi.cap_factor(batch)
    flat = lambda parts: torch.cat([p.reshape(-1) for p in parts])
    deltas = [flat([a[i] for a in (gr, gu, gd)]) for i in (2, 3)]
    if bias:
        deltas += [flat([a[i] for a in (gr, gu, gd)]) for i in (4, 5)]
    for name, p, d in ((names[0], norm, list(gn[2:])), (names[1], moe, deltas)):
        F.param_update(d[0].contiguous(), d[1].contiguous(), cap, p[0], p[1])
        if bias:
            F.param_update(d[2].contiguous(), d[3].contiguous(), cap, p[2], p[3])
        for a, b in zip(_params(net, name), p):
            if a is not None:
                assert torch.equal(a, b), name


def _train(net, cutagi, xs, ys):
    updater = cutagi.OutputUpdater(net.device)
    trace = []
    for x, y in zip(xs, ys):
        net.forward(x)
        trace.append([a.copy() for a in net.get_outputs()])
        updater.update(net.output_z_buffer, y, np.full(y.size, 0.5, np.float32), net.input_delta_z_buffer)
        net.backward()
        net.step()
    return trace, net.state_dict()


def test_replay_gives_the_eager_bits():
    from cutagi_amd import cutagi
    rng = np.random.default_rng(0)
    sizes = [32] * 5 + [9] * 4 + [64] * 4 + [32] * 2
    xs = [rng.standard_normal((b, 16)).astype(np.float32) for b in sizes]
    ys = [rng.standard_normal(b * N_OUT).astype(np.float32) for b in sizes]
    eager, p0 = _train(_net(cutagi), cutagi, xs, ys)
    net = _net(cutagi)
    net.enable_graphs(True)
    replay, p1 = _train(net, cutagi, xs, ys)
    captured = net.graphs_captured()
    net.enable_graphs(False)
    for i, (a, b) in enumerate(zip(eager, replay)):
        assert all(np.array_equal(u, w) for u, w in zip(a, b)), "outputs differ at step %d" % i
    assert p0 == p1 and captured >= 2
    assert all(np.all(np.isfinite(u)) for a in eager for u in a)


@pytest.mark.parametrize("first", ["forward", "eval"])
def test_backward_scratch_that_grows_later_drops_the_recordings(first):
    """1024 features: 100 and 200 rows need different amounts of scratch memory for the layer
    norm's parameter sums, and a pass of 512 rows before them leaves nothing else to grow."""
    from cutagi_amd import capi, cutagi
    assert 0 < capi.layernorm_bwd_scratch(1024, 100) < capi.layernorm_bwd_scratch(1024, 200)
    rng = np.random.default_rng(5)
    sizes = [100] * 5 + [200] + [100] * 5
    xs = [rng.standard_normal((b, 16)).astype(np.float32) for b in sizes]
    ys = [rng.standard_normal(b * N_OUT).astype(np.float32) for b in sizes]
    large = rng.standard_normal((512, 16)).astype(np.float32)

    def run(graphs):
        cutagi.manual_seed(0)
        net = cutagi.Sequential([cutagi.Linear(16, 1024), cutagi.MixtureReLU(), cutagi.LayerNorm([1024]),
                                 cutagi.MixtureOfExperts(1024, 24, N_OUT, 4, 2)])
        net.to_device("cuda")
        net.enable_graphs(graphs)
        if first == "eval":
            net.eval()
        net.forward(large)
        net.train()
        trace, params = _train(net, cutagi, xs, ys)
        captured = net.graphs_captured()
        net.enable_graphs(False)
        return trace, params, captured
    (eager, p0, _), (replay, p1, captured) = run(False), run(True)
    for i, (a, b) in enumerate(zip(eager, replay)):
        assert all(np.array_equal(u, w) for u, w in zip(a, b)), "outputs differ at step %d" % i
    assert p0 == p1 and captured >= 2
    assert all(np.all(np.isfinite(u)) for a in eager for u in a)


def test_expert_choices_after_replays():
    """Of the last pass, replayed or not, whatever batch ran last by itself."""
    from cutagi_amd import cutagi
    rng = np.random.default_rng(6)
    xs = {b: rng.standard_normal((b, 16)).astype(np.float32) for b in (32, 9, 64)}
    eager, net = _net(cutagi), _net(cutagi)
    eager.eval()
    net.eval()
    net.enable_graphs(True)
    net.forward(xs[64])
    for b in [32] * 5 + [9] * 5 + [64, 32, 9, 64, 32, 64, 9, 32]:
        x = xs[b] + rng.standard_normal(xs[b].shape).astype(np.float32)
        net.forward(x)
        eager.forward(x)
        choices = net.layers[3].get_expert_choices()
        assert len(choices) == b * TOP_K
        assert choices == eager.layers[3].get_expert_choices()
    assert net.graphs_captured() >= 2
    net.enable_graphs(False)


@pytest.mark.parametrize("make", ["norm", "experts"])
@pytest.mark.parametrize("graphs", [False, True])
def test_backward_needs_the_forward_pass_of_its_batch(make, graphs):
    """What the two layers keep belongs to the last forward pass: a backward pass after an
    evaluation is refused, and for the experts, whose rows lie elsewhere for every batch, one
    of another batch."""
    from cutagi_amd import cutagi
    cutagi.manual_seed(0)
    last = cutagi.LayerNorm([12]) if make == "norm" else cutagi.MixtureOfExperts(12, 8, 12, 3, 2)
    net = cutagi.Sequential([cutagi.Linear(16, 12), cutagi.MixtureReLU(), last])
    net.to_device("cuda")
    net.enable_graphs(graphs)
    rng = np.random.default_rng(8)
    xs = [rng.standard_normal((10, 16)).astype(np.float32) for _ in range(4)]
    ys = [rng.standard_normal(120).astype(np.float32) for _ in range(4)]
    _train(net, cutagi, xs, ys)
    before = net.state_dict()
    for batch in (10, 4, 20):
        net.forward(xs[0])
        net.eval()
        net.forward(np.resize(xs[1], (batch, 16)))
        net.train()
        with pytest.raises(RuntimeError, match="without its forward pass"):
            net.backward()
    net.forward(xs[0])
    net.input_delta_z_buffer.block_size = 11
    with pytest.raises(RuntimeError, match="without its forward pass"):
        net.backward()
    net.input_delta_z_buffer.block_size = 7
    if make == "experts":
        with pytest.raises(RuntimeError, match="without its forward pass"):
            net.backward()
    assert [n for n in before if before[n] != net.state_dict()[n]] == []
    # and it goes on as if nothing had been
    _, got = _train(net, cutagi, xs, ys)
    net.enable_graphs(False)
    other = cutagi.Sequential([cutagi.Linear(16, 12), cutagi.MixtureReLU(),
                               cutagi.LayerNorm([12]) if make == "norm" else cutagi.MixtureOfExperts(12, 8, 12, 3, 2)])
    other.to_device("cuda")
    other.load_state_dict(before)
    _, want = _train(other, cutagi, xs, ys)
    assert [n for n in want if want[n] != got[n]] == []


def test_residual_block_and_evaluation_mode():
    """x + experts(norm(x)): the block adds the shortcut forward and its innovations back."""
    from cutagi_amd import cutagi
    rng = np.random.default_rng(1)
    cutagi.manual_seed(3)
    block = cutagi.LayerBlock([cutagi.LayerNorm([16]), cutagi.MixtureOfExperts(16, 24, 16, 4, 2)])
    net = cutagi.Sequential([cutagi.Linear(8, 16), cutagi.ResNetBlock(block), cutagi.Linear(16, 3)])
    net.to_device("cuda")
    xs = [rng.standard_normal((10, 8)).astype(np.float32) for _ in range(4)]
    ys = [rng.standard_normal(30).astype(np.float32) for _ in range(4)]
    trace, _ = _train(net, cutagi, xs, ys)
    assert all(np.all(np.isfinite(u)) for a in trace for u in a)
    # against the layers one by one, with the sum in between
    net.eval()
    net.forward(xs[0])
    got = [np.asarray(a) for a in net.get_outputs()]
    import torch
    import cutagi_amd.functional as F
    sd = net.state_dict()
    p = lambda n: [torch.tensor(a, dtype=torch.float32, device="cuda") for a in sd[n]]
    keys = {k.split(".")[0] + "." + k.rsplit(".", 1)[-1]: k for k in sd}
    lin0, lin2 = sorted(k for k in sd if k.startswith("Linear"))
    ln = next(k for k in sd if "LayerNorm" in k)
    me = next(k for k in sd if "MixtureOfExperts" in k)
    a = torch.from_numpy(xs[0]).cuda()
    w = p(lin0)
    h = F.linear_fwd(w[0].reshape(16, 8), w[1].reshape(16, 8), w[2], w[3], a, torch.zeros_like(a))
    z = F.layernorm_fwd(*p(ln), *h, 1e-5)
    q = p(me)
    E, K, H, N = 4, 16, 24, 16
    part = lambda x, a, n, s: x[a:a + n].reshape(s).clone()
    wr = [part(x, 0, E * K, (E, K)) for x in q[:2]] + [part(x, 0, E, (E,)) for x in q[2:]]
    wu = [part(x, E * K, E * H * K, (E, H, K)) for x in q[:2]] + [part(x, E, E * H, (E, H)) for x in q[2:]]
    wd = [part(x, E * K + E * H * K, E * N * H, (E, N, H)) for x in q[:2]] + [part(x, E + E * H, E * N, (E, N)) for x in q[2:]]
    r = F.moe_route(*F.linear_fwd(*wr, z[0], z[1]), 2)
    u = F.grouped_linear_fwd_act(*wu, z[0], z[1], r.offsets, "relu", rows=r.token)
    y = F.grouped_linear_fwd(*wd, u[0], u[1], r.offsets)
    c = F.moe_combine_fwd(r.mu_g, r.var_g, *y, r.slot)
    w = p(lin2)
    want = F.linear_fwd(w[0].reshape(3, 16), w[1].reshape(3, 16), w[2], w[3], c[0] + h[0], c[1] + h[1])
    for g, x in zip(got, want):
        assert np.array_equal(g.ravel(), x.cpu().numpy().ravel()), keys


@pytest.mark.parametrize("shortcut", [False, True])
@pytest.mark.parametrize("batch", [10, 300])
def test_training_through_a_residual_block_is_its_calls(batch, shortcut):
    """Steps of x + experts(norm(x)) behind an activation, whose Jacobian meets the innovations of
    both branches: every parameter has the bits of the tensor-level calls, step after step."""
    import torch
    import cutagi_amd.functional as F
    from cutagi_amd import capi, cutagi
    cutagi.manual_seed(12)
    branch = [cutagi.LayerBlock([cutagi.Linear(N_IN, 20), cutagi.ReLU(), cutagi.Linear(20, N_IN)])] if shortcut else []
    block = cutagi.LayerBlock([cutagi.LayerNorm([N_IN]), cutagi.MixtureOfExperts(N_IN, HIDDEN, N_IN, EXPERTS, TOP_K)])
    net = cutagi.Sequential([cutagi.Linear(8, N_IN), cutagi.MixtureReLU(), cutagi.ResNetBlock(block, *branch),
                             cutagi.Linear(N_IN, 3)])
    net.to_device("cuda")
    rng = np.random.default_rng(batch)
    xs = [rng.standard_normal((batch, 8)).astype(np.float32) for _ in range(3)]
    ys = [rng.standard_normal(batch * 3).astype(np.float32) for _ in range(3)]
    names = {part: next(k for k in net.state_dict() if part in k)
             for part in ("LinearCuda.0", "LayerNorm", "MixtureOfExperts", "LinearCuda.3")}
    if shortcut:
        names.update({"sc%d" % i: "LinearCuda.shortcut.2.%d" % i for i in (0, 2)})
    p = {part: _params(net, name) for part, name in names.items()}
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()

    def linear(part, N, K):
        m, v, b, q = p[part]
        return m.view(N, K), v.view(N, K), b, q

    for x, y in zip(xs, ys):
        a, zero = t(x), torch.zeros(batch, 8, device="cuda")
        h, vh, jh = F.linear_fwd_act(*linear("LinearCuda.0", N_IN, 8), a, zero, "mixture_relu")
        z, vz, m, s = F.layernorm_fwd(*p["LayerNorm"], h, vh, 1e-5)
        parts = _split_square(p["MixtureOfExperts"])
        router, up, down = parts
        r = F.moe_route(*F.linear_fwd(*router, z, vz), TOP_K)
        g, vg, jg = F.grouped_linear_fwd_act(*up, z, vz, r.offsets, "relu", rows=r.token)
        e, ve = F.grouped_linear_fwd(*down, g, vg, r.offsets)
        c, vc = F.moe_combine_fwd(r.mu_g, r.var_g, e, ve, r.slot)
        if shortcut:
            k, vk, jk = F.linear_fwd_act(*linear("sc0", 20, N_IN), h, vh, "relu")
            F.add_shortcut(*F.linear_fwd(*linear("sc2", N_IN, 20), k, vk), c, vc)
        else:
            F.add_shortcut(h, vh, c, vc)
        o, vo = F.linear_fwd(*linear("LinearCuda.3", 3, N_IN), c, vc)
        net.forward(x)
        for got, want in zip(net.get_outputs(), (o, vo)):
            assert np.array_equal(np.asarray(got).ravel(), _host_flat(want))

        one = torch.ones_like
        dmu, dvar = torch.zeros_like(o), torch.zeros_like(o)
        F.out_update_dense(o, vo, one(o), t(y), torch.full((batch * 3,), 0.5, device="cuda"), dmu, dvar)
        w = linear("LinearCuda.3", 3, N_IN)
        last = F.linear_bwd(w[0], w[1], w[3], c, one(c), dmu, dvar)
        do = last[:2]
        d = {"LinearCuda.3": last[2:]}
        de, dve, ds, dvs = F.moe_combine_bwd(r.mu_g, r.jcb_g, e, r.expert, r.slot, *do, EXPERTS)
        gd = F.grouped_linear_bwd(down[0], down[1], down[3], g, jg, de, dve, r.offsets)
        gu = F.grouped_linear_bwd(up[0], up[1], up[3], z, None, gd[0], gd[1], r.offsets, rows=r.token)
        gr = F.linear_bwd(router[0], router[1], router[3], z, one(z), ds, dvs)
        dz = F.moe_gather_bwd(gu[0], gu[1], r.slot, None, gr[0], gr[1])
        d["MixtureOfExperts"] = [torch.cat([q[i].reshape(-1) for q in (gr, gu, gd)]) for i in range(2, 6)]
        norm = F.layernorm_bwd(p["LayerNorm"][0], p["LayerNorm"][1], p["LayerNorm"][3], h, jh, m, s, *dz, 1e-5)
        d["LayerNorm"] = norm[2:]
        dh = norm[:2]
        if shortcut:
            w = linear("sc2", N_IN, 20)
            b2 = F.linear_bwd(w[0], w[1], w[3], k, jk, *do)
            w = linear("sc0", 20, N_IN)
            b0 = F.linear_bwd(w[0], w[1], w[3], h, jh, b2[0], b2[1])
            d["sc2"], d["sc0"] = b2[2:], b0[2:]
            F.add_shortcut(b0[0], b0[1], *dh)
        else:
            F.add_shortcut_delta(*do, jh, *dh)
        w = linear("LinearCuda.0", N_IN, 8)
        d["LinearCuda.0"] = F.linear_bwd(w[0], w[1], w[3], a, one(a), *dh, state_update=False)[2:]
        cap = capi.cap_factor(batch)
        for part, (m_w, v_w, m_b, v_b) in d.items():
            F.param_update(m_w.reshape(-1), v_w.reshape(-1), cap, p[part][0], p[part][1])
            F.param_update(m_b.reshape(-1), v_b.reshape(-1), cap, p[part][2], p[part][3])

        updater = cutagi.OutputUpdater(net.device)
        updater.update(net.output_z_buffer, y, np.full(y.size, 0.5, np.float32), net.input_delta_z_buffer)
        net.backward()
        net.step()
        for part, name in names.items():
            for i, (got, want) in enumerate(zip(_params(net, name), p[part])):
                assert torch.equal(got, want), "%s, array %d" % (name, i)


def _host_flat(t):
    return t.cpu().numpy().ravel()


def _split_square(p):
    """_split for experts that put out as many features as they take."""
    E, K, H = EXPERTS, N_IN, HIDDEN
    ends, bends = [0, E * K, E * K + E * H * K, E * K + 2 * E * H * K], [0, E, E + E * H, E + E * H + E * K]
    shapes, bshapes = [(E, K), (E, H, K), (E, K, H)], [(E,), (E, H), (E, K)]
    return [[x[ends[i]:ends[i + 1]].view(shapes[i]) for x in p[:2]] +
            [x[bends[i]:bends[i + 1]].view(bshapes[i]) for x in p[2:]] for i in range(3)]


def test_two_blocks_through_the_python_layer():
    """Blocks one behind the other, batches of different sizes: finite, and a step moves every
    layer's parameters."""
    from cutagi_amd import cutagi
    from cutagi_amd.nn import (LayerBlock, LayerNorm, Linear, MixtureOfExperts, OutputUpdater, ReLU, ResNetBlock,
                               Sequential)
    cutagi.manual_seed(3)
    experts = lambda: ResNetBlock(LayerBlock(LayerNorm(64), MixtureOfExperts(64, 256, 64, num_experts=8, top_k=2)))
    net = Sequential(Linear(32, 64), ReLU(), experts(), experts(), LayerNorm(64), Linear(64, 10))
    net.to_device("cuda")
    updater = OutputUpdater(net.device)
    rng = np.random.default_rng(3)
    before = net.state_dict()
    for batch in (16, 3, 64, 16):
        mu, var = net(rng.standard_normal(batch * 32).astype(np.float32))
        assert np.all(np.isfinite(mu)) and np.all(np.asarray(var) > 0)
        updater.update(net.output_z_buffer, rng.standard_normal(batch * 10).astype(np.float32),
                       np.full(batch * 10, 0.5, np.float32), net.input_delta_z_buffer)
        net.backward()
        net.step()
    after = net.state_dict()
    assert sorted(after) == sorted(before) and len(after) >= 6
    for name in after:
        for a, b in zip(after[name], before[name]):
            assert len(a) == len(b) and np.all(np.isfinite(a))
            assert len(a) == 0 or np.any(np.asarray(a) != np.asarray(b)), name


@pytest.mark.parametrize("features", [16, 64])
def test_residual_block_of_features_behind_an_image(features):
    """More and fewer features than the image has pixels: the same bits as from the block by
    itself, given what the layers before it put out."""
    from cutagi_amd import cutagi
    rng = np.random.default_rng(10)
    cutagi.manual_seed(4)
    block = lambda: cutagi.ResNetBlock(cutagi.LayerBlock([cutagi.LayerNorm([features]),
                                                          cutagi.MixtureOfExperts(features, 24, features, 4, 2)]))
    head = lambda: [cutagi.Conv2d(1, 2, 3, padding=1, in_width=4, in_height=4), cutagi.ReLU(),
                    cutagi.Linear(32, features)]
    net, first, second = (cutagi.Sequential(layers) for layers in (head() + [block()], head(), [block()]))
    for n in (net, first, second):
        n.to_device("cuda")
        n.preinit_layer()
    sd = net.state_dict()
    first.load_state_dict({k: v for k, v in sd.items() if "main" not in k})
    second.load_state_dict({k.replace("main.3", "main.0"): v for k, v in sd.items() if "main" in k})
    x = rng.standard_normal((10, 16)).astype(np.float32)
    net.forward(x)
    first.forward(x)
    second.forward(*first.get_outputs())
    got, want = net.get_outputs(), second.get_outputs()
    assert got[0].size == 10 * features
    assert all(np.array_equal(a, b) for a, b in zip(got, want))
    before = net.state_dict()
    _train(net, cutagi, [x] * 2, [rng.standard_normal(10 * features).astype(np.float32)] * 2)
    after = net.state_dict()
    assert all(np.all(np.isfinite(a)) for p in after.values() for a in p)
    assert [k for k in after if after[k] == before[k]] == []


def test_checkpoints(tmp_path):
    from cutagi_amd import cutagi
    net, other = _net(cutagi, seed=0), _net(cutagi, seed=1)
    x = np.random.default_rng(0).standard_normal((5, 16)).astype(np.float32)
    net.forward(x)
    want = [a.copy() for a in net.get_outputs()]
    other.forward(x)
    assert not np.array_equal(want[0], other.get_outputs()[0])
    net.save(str(tmp_path / "net.bin"))
    other.load(str(tmp_path / "net.bin"))
    assert net.state_dict() == other.state_dict()
    other.forward(x)
    assert all(np.array_equal(a, b) for a, b in zip(want, other.get_outputs()))
    third = _net(cutagi, seed=2)
    third.load_state_dict(net.state_dict())
    third.forward(x)
    assert all(np.array_equal(a, b) for a, b in zip(want, third.get_outputs()))


@pytest.mark.parametrize("where", ["device", "host", "model"])
def test_parameters_of_other_sizes_are_refused(where):
    """A state dict, or a model, of layers with other sizes under the same names: the forward
    pass raises, and the right parameters put it right again."""
    from cutagi_amd import cutagi
    x = np.zeros((3, 12), np.float32)

    def make(norm, experts, hidden=8, bias=True, device=True):
        cutagi.manual_seed(0)
        net = cutagi.Sequential([cutagi.LayerNorm([norm], 1e-5, bias),
                                 cutagi.MixtureOfExperts(norm, hidden, 12, experts, 2, "relu", bias)])
        if device:
            net.to_device("cuda")
        return net
    for wrong in (make(10, 3), make(12, 2), make(12, 3, hidden=7), make(14, 3), make(12, 3, bias=False)):
        net = make(12, 3, device=where != "host")
        right = net.state_dict()
        if where == "model":
            net.params_from(wrong)
        elif where == "device":
            net.load_state_dict(wrong.state_dict())
        else:
            net.load_state_dict({k.replace("Cuda", ""): v for k, v in wrong.state_dict().items()})
            net.to_device("cuda")
        with pytest.raises(RuntimeError, match="expected"):
            net.forward(x)
        net.load_state_dict({(k if "Cuda" in k else k.replace(".", "Cuda.")): v for k, v in right.items()})
        net.forward(x)
        assert all(np.all(np.isfinite(a)) for a in net.get_outputs())


def test_refusals():
    from cutagi_amd import cutagi
    net = _net(cutagi, first=False)
    with pytest.raises(RuntimeError, match="mismatch"):
        net.forward(np.zeros((2, N_IN + 1), np.float32))
    bad = cutagi.Sequential([cutagi.Linear(4, 6), cutagi.LayerNorm([8])])
    bad.to_device("cuda")
    with pytest.raises(RuntimeError, match="mismatch"):
        bad.forward(np.zeros((2, 4), np.float32))
