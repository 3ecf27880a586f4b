"""HIP graph replay of a Sequential's forward / backward passes (enable_graphs):
the same training run with replay on and off gives the same bits, step after step,
through batch-size changes, mode switches and parameter reloads; the replays are
separated by the eager parts of a step (input transfer, output update, parameter
update, output read-back with its synchronisation), as they are in use."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _mlp(cutagi):
    cutagi.manual_seed(0)
    net = cutagi.Sequential([cutagi.Linear(784, 128), cutagi.ReLU(), cutagi.Linear(128, 128),
                             cutagi.ReLU(), cutagi.Linear(128, 11)])
    net.to_device("cuda")
    return net


def _cnn(cutagi):
    cutagi.manual_seed(1)
    net = cutagi.Sequential([
        cutagi.Conv2d(3, 8, 3, bias=False, padding=1, in_width=8, in_height=8), cutagi.MixtureReLU(),
        cutagi.BatchNorm2d(8), cutagi.Conv2d(8, 8, 3, bias=True, stride=2, padding=1, padding_type=2),
        cutagi.ReLU(), cutagi.AvgPool2d(2, 2), cutagi.Linear(8 * 2 * 2, 5)])
    net.to_device("cuda")
    net.preinit_layer()
    return net


def _train(net, cutagi, xs, ys, n_out, observe=None):
    updater = cutagi.OutputUpdater(net.device)
    trace = []
    for step, (x, y) in enumerate(zip(xs, ys)):
        if observe is not None:
            observe(step, net)
        net.forward(x)
        mu, var = net.get_outputs()
        updater.update(net.output_z_buffer, y, np.full(y.size, 0.5, np.float32),
                       net.input_delta_z_buffer)
        net.backward()
        net.step()
        trace.append((mu.copy(), var.copy()))
    return trace, net.state_dict()


@pytest.mark.parametrize("make,n_in,n_out", [(_mlp, 784, 11), (_cnn, 3 * 8 * 8, 5)])
def test_replay_gives_the_eager_bits(make, n_in, n_out):
    from cutagi_amd import cutagi
    rng = np.random.default_rng(0)
    # the batch size changes twice; every size is seen often enough to be recorded
    sizes = [32] * 6 + [16] * 5 + [32] * 4
    xs = [rng.normal(0, 1, (b, n_in)).astype(np.float32) for b in sizes]
    ys = [rng.normal(0, 1, b * n_out).astype(np.float32) for b in sizes]
    eager_net = make(cutagi)
    eager, eager_params = _train(eager_net, cutagi, xs, ys, n_out)
    net = make(cutagi)
    net.enable_graphs(True)
    assert net.graphs_enabled()
    captured = []
    replay, replay_params = _train(net, cutagi, xs, ys, n_out,
                                   observe=lambda s, n: captured.append(n.graphs_captured()))
    for s, ((m0, v0), (m1, v1)) in enumerate(zip(eager, replay)):
        assert np.array_equal(m0, m1) and np.array_equal(v0, v1), "outputs differ at step %d" % s
    assert eager_params == replay_params
    # two eager runs per key, then a forward and a backward graph for batch 32, later for 16
    assert captured[2] == 0 and captured[4] == 2 and max(captured) >= 4
    net.enable_graphs(False)
    assert net.graphs_captured() == 0


def test_mode_switches_and_reloads_drop_the_recordings():
    from cutagi_amd import cutagi
    rng = np.random.default_rng(1)
    net = _mlp(cutagi)
    net.enable_graphs(True)
    twin = _mlp(cutagi)
    x = rng.normal(0, 1, (8, 784)).astype(np.float32)
    y = rng.normal(0, 1, 8 * 11).astype(np.float32)
    _train(net, cutagi, [x] * 5, [y] * 5, 11)
    _train(twin, cutagi, [x] * 5, [y] * 5, 11)
    assert net.graphs_captured() == 2
    net.eval()
    assert net.graphs_captured() == 0
    twin.eval()
    for _ in range(4):      # eval-mode forwards: eager twice, then recorded, same outputs
        net.forward(x)
        twin.forward(x)
        assert np.array_equal(net.get_outputs()[0], twin.get_outputs()[0])
    assert net.graphs_captured() == 1
    net.train()
    twin.train()
    # other parameters under a recorded graph: the recording must not survive the reload
    other = _mlp(cutagi)
    _train(other, cutagi, [x] * 2, [y] * 2, 11)
    sd = other.state_dict()
    net.load_state_dict(sd)
    twin.load_state_dict(sd)
    assert net.graphs_captured() == 0
    a, pa = _train(net, cutagi, [x] * 5, [y] * 5, 11)
    b, pb = _train(twin, cutagi, [x] * 5, [y] * 5, 11)
    assert all(np.array_equal(p[0], q[0]) for p, q in zip(a, b)) and pa == pb


def _eager_and_replayed(make, cutagi, steps, n_in, n_out):
    """Runs `steps` - ("train" | "indexed" | "forward", batch) or "eval" / "train" - on a network with
    graphs and on one without, and compares outputs and parameters. Returns the graphs held
    before every step."""
    rng = np.random.default_rng(4)
    data = [s if isinstance(s, str) else
            (s[0], rng.normal(0, 1, (s[1], n_in)).astype(np.float32),
             rng.normal(0, 1, s[1] * n_out).astype(np.float32)) for s in steps]
    held = []

    def run(net, note):
        updater = cutagi.OutputUpdater(net.device)
        trace = []
        for s in data:
            if note:
                held.append(net.graphs_captured())
            if isinstance(s, str):
                getattr(net, s)()
                continue
            kind, x, y = s
            net.forward(x)
            trace.append([a.copy() for a in net.get_outputs()])
            if kind == "train":
                updater.update(net.output_z_buffer, y, np.full(y.size, 0.5, np.float32),
                               net.input_delta_z_buffer)
            elif kind == "indexed":      # two observed outputs per sample
                idx = np.tile(np.array([1, n_out], np.int32), len(x))
                updater.update_using_indices(net.output_z_buffer, y[:2 * len(x)],
                                             np.full(2 * len(x), 0.5, np.float32), idx,
                                             net.input_delta_z_buffer)
            if kind != "forward":
                net.backward()
                net.step()
        return trace, net.state_dict()
    eager, eager_params = run(make(cutagi), False)
    net = make(cutagi)
    net.enable_graphs(True)
    replay, replay_params = run(net, True)
    net.enable_graphs(False)
    for i, (a, b) in enumerate(zip(eager, replay)):
        assert all(np.array_equal(u, w) for u, w in zip(a, b)), "outputs differ at step %d" % i
    assert all(np.all(np.isfinite(u)) for a in eager for u in a)
    differ = [name for name in eager_params if eager_params[name] != replay_params[name]]
    assert not differ
    return held


@pytest.mark.parametrize("make,n_in,n_out", [(_mlp, 784, 11), (_cnn, 3 * 8 * 8, 5)])
def test_training_buffers_that_grow_later_drop_the_recordings(make, n_in, n_out):
    """An evaluation of a larger batch first: the state buffers do not grow with the training
    batches any more, but what the layers keep for the backward pass does."""
    from cutagi_amd import cutagi
    steps = ["eval", ("forward", 256), "train"] + [("train", b) for b in [32] * 5 + [64] * 2 + [32] * 5 + [64] * 4]
    held = _eager_and_replayed(make, cutagi, steps, n_in, n_out)
    assert held[7] == 2      # recorded at 32
    assert held[9] == 0      # after the first step at 64: dropped
    assert max(held[10:]) >= 2


@pytest.mark.parametrize("make,n_in,n_out", [(_mlp, 784, 11), (_cnn, 3 * 8 * 8, 5)])
def test_replayed_batches_are_capped_by_their_own_size(make, n_in, n_out):
    """The cap of the parameter updates depends on the batch: one sample, up to 255, more."""
    from cutagi_amd import cutagi
    sizes = [300] * 5 + [32] * 5 + [300] * 2 + [1] * 5 + [32] * 2 + [1, 300, 1]
    held = _eager_and_replayed(make, cutagi, [("train", b) for b in sizes], n_in, n_out)
    assert max(held) >= 6


def _even(cutagi):
    """Two passes: the output lies in the object that the input was written to."""
    cutagi.manual_seed(3)
    net = cutagi.Sequential([cutagi.Linear(24, 16), cutagi.ReLU(), cutagi.Linear(16, 6)])
    net.to_device("cuda")
    return net


@pytest.mark.parametrize("make,n_in,n_out", [(_even, 24, 6), (_mlp, 784, 11), (_cnn, 3 * 8 * 8, 5)])
def test_indexed_update_after_a_replay(make, n_in, n_out):
    """The update finds the outputs of a sample by the size that the forward pass gave them."""
    from cutagi_amd import cutagi
    sizes = [32] * 9 + [16] * 9 + [32] * 3 + [16] * 2
    held = _eager_and_replayed(make, cutagi, [("indexed", b) for b in sizes], n_in, n_out)
    assert max(held) >= 4


def _experts(cutagi):
    cutagi.manual_seed(5)
    net = cutagi.Sequential([cutagi.Linear(12, 20), cutagi.MixtureReLU(), cutagi.LayerNorm([20]),
                             cutagi.MixtureOfExperts(20, 24, 6, 4, 2)])
    net.to_device("cuda")
    return net


def _residual(cutagi):
    cutagi.manual_seed(6)
    block = cutagi.LayerBlock([cutagi.LayerNorm([20]), cutagi.MixtureOfExperts(20, 24, 20, 4, 2)])
    net = cutagi.Sequential([cutagi.Linear(12, 20), cutagi.ResNetBlock(block), cutagi.Linear(20, 6)])
    net.to_device("cuda")
    return net


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("make,n_in,n_out", [(_mlp, 784, 11), (_cnn, 3 * 8 * 8, 5), (_experts, 12, 6),
                                             (_residual, 12, 6)])
def test_evaluations_between_training_steps_leave_the_steps_alone(make, n_in, n_out, graphs):
    """An evaluation of another batch size, smaller or larger, and training steps of the size
    of that evaluation: the same parameters as without the evaluations."""
    from cutagi_amd import cutagi
    rng = np.random.default_rng(7)
    sizes = [32, 32, 16, 64, 64, 64, 64, 9, 64, 32]
    data = [(rng.normal(0, 1, (b, n_in)).astype(np.float32), rng.normal(0, 1, b * n_out).astype(np.float32))
            for b in sizes]
    other = rng.normal(0, 1, (200, n_in)).astype(np.float32)

    def run(evaluate):
        net = make(cutagi)
        net.enable_graphs(graphs)
        updater = cutagi.OutputUpdater(net.device)
        for i, (x, y) in enumerate(data):
            net.forward(x)
            updater.update(net.output_z_buffer, y, np.full(y.size, 0.5, np.float32), net.input_delta_z_buffer)
            net.backward()
            net.step()
            if evaluate and i + 1 < len(sizes):
                net.eval()
                net.forward(other[:7])
                net.forward(other[:sizes[i + 1]])
                net.train()
        net.enable_graphs(False)
        return net.state_dict()
    plain, evaluated = run(False), run(True)
    differ = [name for name in plain if plain[name] != evaluated[name]]
    assert not differ
    assert all(np.all(np.isfinite(a)) for p in plain.values() for a in p)


def _conv_block(cutagi):
    cutagi.manual_seed(7)
    block = lambda: cutagi.LayerBlock([cutagi.Conv2d(2, 2, 3, padding=1, in_width=4, in_height=4), cutagi.ReLU(),
                                       cutagi.Conv2d(2, 2, 3, padding=1)])
    res = [cutagi.ResNetBlock(block()), cutagi.ResNetBlock(block(), block())]
    res[0].in_width, res[0].in_height, res[0].in_channels = 4, 4, 2
    net = cutagi.Sequential(res + [cutagi.Linear(32, 6)])
    net.to_device("cuda")
    net.preinit_layer()      # (the convolutions draw their weights here, not in the first pass)
    return net


@pytest.mark.parametrize("make,n_in", [(_residual, 12), (_conv_block, 32)])
def test_blocks_refuse_a_backward_pass_after_an_evaluation(make, n_in):
    """The first layers of a block borrow the input that it keeps, and an evaluation puts its
    own there."""
    from cutagi_amd import cutagi
    rng = np.random.default_rng(9)
    xs = [rng.normal(0, 1, (10, n_in)).astype(np.float32) for _ in range(3)]
    ys = [rng.normal(0, 1, 60).astype(np.float32) for _ in range(3)]
    net, twin = make(cutagi), make(cutagi)
    _train(net, cutagi, xs, ys, 6)
    for batch in (10, 4, 20):
        net.forward(xs[0])
        net.eval()
        net.forward(np.resize(xs[1], (batch, n_in)))
        net.train()
        with pytest.raises(RuntimeError, match="without its forward pass"):
            net.backward()
    _train(twin, cutagi, xs, ys, 6)
    (_, got), (_, want) = (_train(n, cutagi, xs, ys, 6) for n in (net, twin))
    assert [n for n in want if want[n] != got[n]] == []


def test_workspace_of_a_recorded_call_outlives_its_growth():
    """A sliced reduction recorded with the workspace of its stream, which then grows: the
    recording still owns the memory that its partial sums go to."""
    import torch
    import cutagi_amd.functional as F
    from cutagi_amd import capi
    torch.cuda.synchronize()
    capi.check(capi.lib.tagi_hip_shutdown())
    K, N, B = 4096, 2048, 256        # eight reduction slices: 32 MiB of partial sums
    mk = lambda *s: torch.rand(*s, device="cuda")
    w, v, a, q = mk(N, K) - 0.5, mk(N, K), mk(B, K), mk(B, K)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    free = [torch.cuda.mem_get_info()[0]]
    with torch.cuda.stream(stream):
        want = F.linear_fwd(w, v, None, None, a, q)
    stream.synchronize()
    free.append(torch.cuda.mem_get_info()[0])
    assert free[0] - free[1] > 16 << 20, "no workspace grew"
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = F.linear_fwd(w, v, None, None, a, q)
    free.append(torch.cuda.mem_get_info()[0])
    capi.check(capi.lib.tagi_hip_workspace_reserve(1 << 30, stream.cuda_stream))
    # 1 GiB where the old 32 MiB are kept, 32 MiB less where not (the runtime moves some pages
    # of 2 MiB by itself: the limit lies halfway)
    assert free[2] - torch.cuda.mem_get_info()[0] > (1 << 30) - (16 << 20), "the outgrown workspace was freed"
    other = torch.full((64 << 20,), float("nan"), device="cuda")     # would lie where it was
    for i in range(3):
        a.mul_(1.01)
        with torch.cuda.stream(stream):
            stream.wait_stream(torch.cuda.default_stream())
            want = F.linear_fwd(w, v, None, None, a, q)
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), "replay %d" % i
    assert bool(torch.isnan(other).all())
    del graph
    free.append(torch.cuda.mem_get_info()[0])
    capi.check(capi.lib.tagi_hip_shutdown())
    assert torch.cuda.mem_get_info()[0] - free[3] > (1 << 30) + (16 << 20)


def test_networks_with_blocks_stay_eager():
    from cutagi_amd import cutagi
    cutagi.manual_seed(2)
    block = cutagi.LayerBlock([cutagi.Conv2d(2, 2, 3, padding=1, in_width=4, in_height=4),
                               cutagi.ReLU(), cutagi.Conv2d(2, 2, 3, padding=1)])
    res = cutagi.ResNetBlock(block)
    res.in_width, res.in_height, res.in_channels = 4, 4, 2
    net = cutagi.Sequential([res, cutagi.Linear(32, 3)])
    net.to_device("cuda")
    net.enable_graphs(True)
    rng = np.random.default_rng(2)
    x = rng.normal(0, 1, (4, 32)).astype(np.float32)
    y = rng.normal(0, 1, 12).astype(np.float32)
    trace, _ = _train(net, cutagi, [x] * 5, [y] * 5, 3)
    assert net.graphs_captured() == 0 and all(np.all(np.isfinite(m)) for m, _ in trace)
