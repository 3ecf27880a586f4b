"""Refusals of the layer norm, grouped Linear and mixture-of-experts entry points, without a
GPU: argument checks come before any launch."""
import ctypes

import pytest
import torch

one = ctypes.c_void_p(16)   # never dereferenced: the checks fire first
odd = ctypes.c_void_p(20)


def _lib():
    from cutagi_amd import capi
    return capi, capi.lib


def _without(args, i, value=None):
    return args[:i] + [value] + args[i + 1:]


def test_layernorm_refuses():
    capi, L = _lib()
    fwd = [one] * 6 + [1, 1e-5, 8, 4] + [one] * 4 + [None]
    for i in [0, 1, 2, 3, 4, 5, 10, 11, 12, 13]:
        assert L.tagi_layernorm_fwd(*_without(fwd, i)) == capi.ERR_INVALID_ARG
    for n, B in ((1, 4), (0, 4), (8, 0), (8, -1)):     # one feature has no sample variance
        assert L.tagi_layernorm_fwd(*(fwd[:8] + [n, B] + fwd[10:])) == capi.ERR_INVALID_ARG
    bwd = [one] * 9 + [1e-5, 8, 999, 1, 1, 1] + [one] * 7 + [None]
    assert capi.layernorm_bwd_scratch(8, 999) > 0
    for i in [0, 1, 2, 3, 5, 6, 7, 8] + list(range(15, 22)):
        assert L.tagi_layernorm_bwd(*_without(bwd, i)) == capi.ERR_INVALID_ARG
    assert L.tagi_layernorm_bwd(*_without(bwd, 15, odd)) == capi.ERR_INVALID_ARG
    assert L.tagi_layernorm_bwd(*_without(bwd, 10, 1)) == capi.ERR_INVALID_ARG
    size = ctypes.c_size_t(0)
    assert L.tagi_layernorm_bwd_scratch(8, 4, None) == capi.ERR_INVALID_ARG
    assert L.tagi_layernorm_bwd_scratch(1, 4, ctypes.byref(size)) == capi.ERR_INVALID_ARG
    for n, B in ((8, (1 << 30) + 1), ((1 << 30) + 1, 8)):
        assert L.tagi_layernorm_fwd(*(fwd[:8] + [n, B] + fwd[10:])) == capi.ERR_UNSUPPORTED
        assert L.tagi_layernorm_bwd(*(bwd[:10] + [n, B] + bwd[12:])) == capi.ERR_UNSUPPORTED
        assert L.tagi_layernorm_bwd_scratch(n, B, ctypes.byref(size)) == capi.ERR_UNSUPPORTED
    # nothing asked for: done
    assert L.tagi_layernorm_bwd(*([one] * 9 + [1e-5, 8, 4, 1, 0, 0] + [None] * 8)) == capi.OK


def test_layernorm_scratch():
    """What is held for a batch does for every smaller one."""
    capi, _ = _lib()
    for n in (2, 24, 300, 1023, 4096, 9001):
        held = 0
        for B in list(range(1, 2100)) + [4096, 9660, 65536, 1 << 20]:
            now = capi.layernorm_bwd_scratch(n, B)
            assert now >= held
            held = now
    assert capi.layernorm_bwd_scratch(4096, 16) == 0


def test_grouped_linear_refuses():
    capi, L = _lib()
    fwd = [one] * 8 + [8, 8, 4, 16, 16, 1] + [one] * 3 + [None]
    for i in [0, 1, 2, 3, 4, 5, 6, 15, 16]:
        assert L.tagi_grouped_linear_fwd(*_without(fwd, i)) == capi.ERR_INVALID_ARG
    for i in [8, 9, 10, 11, 12]:
        for bad in (0, -3):
            assert L.tagi_grouped_linear_fwd(*_without(fwd, i, bad)) == capi.ERR_INVALID_ARG
    assert L.tagi_grouped_linear_fwd(*_without(fwd, 10, 1025)) == capi.ERR_UNSUPPORTED
    act = [one] * 8 + [8, 8, 4, 16, 16, 1, 1] + [one] * 4 + [None]
    for bad in (0, 3, -1):
        assert L.tagi_grouped_linear_fwd_act(*_without(act, 14, bad)) == capi.ERR_INVALID_ARG
    assert L.tagi_grouped_linear_fwd_act(*_without(act, 18)) == capi.ERR_INVALID_ARG
    bwd = [one] * 9 + [8, 8, 4, 16, 16, 1, 1, 1] + [one] * 7 + [None]
    for i in [0, 1, 2, 3, 5, 6, 7] + list(range(18, 24)):
        assert L.tagi_grouped_linear_bwd(*_without(bwd, i)) == capi.ERR_INVALID_ARG
    assert L.tagi_grouped_linear_bwd(*_without(bwd, 11, 2000)) == capi.ERR_UNSUPPORTED
    # more tiles than a launch holds
    huge = [one] * 8 + [1 << 30, 1 << 30, 1024, 16, 16, 1] + [one] * 3 + [None]
    assert L.tagi_grouped_linear_fwd(*huge) == capi.ERR_UNSUPPORTED
    huge = [one] * 9 + [1 << 30, 1 << 30, 1024, 16, 16, 1, 0, 1] + [one] * 7 + [None]
    assert L.tagi_grouped_linear_bwd(*huge) == capi.ERR_UNSUPPORTED
    # more threads than a launch holds: weights in pieces of 32 x 256, rows of one or two inputs
    huge = [one] * 9 + [4, 1 << 24, 1024, 16, 16, 1, 0, 1] + [one] * 7 + [None]
    assert L.tagi_grouped_linear_bwd(*huge) == capi.ERR_UNSUPPORTED
    huge = [one] * 8 + [1, 1, 4, 1 << 28, 16, 1] + [one] * 3 + [None]
    assert L.tagi_grouped_linear_fwd(*huge) == capi.ERR_UNSUPPORTED
    # scratch that is needed and missing, or not 16-byte aligned
    size = capi.grouped_linear_scratch(256, 128, 4, 400)
    assert size > 0
    for scratch in (None, odd):
        call = _without(_without(fwd, 11, 400), 14, scratch)
        assert L.tagi_grouped_linear_fwd(*call) == capi.ERR_INVALID_ARG
        call = _without(_without(bwd, 12, 400), 17, scratch)
        assert L.tagi_grouped_linear_bwd(*call) == capi.ERR_INVALID_ARG


def test_grouped_linear_scratch():
    capi, L = _lib()
    size = ctypes.c_size_t(0)
    for bad in ((0, 8, 4, 16), (8, -1, 4, 16), (8, 8, 0, 16), (8, 8, 4, 0)):
        assert L.tagi_grouped_linear_scratch(*bad, ctypes.byref(size)) == capi.ERR_INVALID_ARG
    assert L.tagi_grouped_linear_scratch(8, 8, 4, 16, None) == capi.ERR_INVALID_ARG
    assert L.tagi_grouped_linear_scratch(8, 8, 1025, 16, ctypes.byref(size)) == capi.ERR_UNSUPPORTED
    assert capi.grouped_linear_scratch(4096, 4096, 8, 8) == 0
    # what is held for a batch does for every smaller one
    for K, N, E in ((64, 48, 4), (2048, 4096, 8), (3, 100, 2), (515, 20, 2), (4100, 300, 1)):
        held = 0
        for R in list(range(1, 300)) + [1000, 4096, 8192, 100000, 1 << 20]:
            now = capi.grouped_linear_scratch(K, N, E, R)
            assert now >= held
            held = now
    assert held < 1 << 26


def test_router_refuses():
    capi, L = _lib()
    route = [one, one, 300, 8, 2] + [one] * 8 + [None]
    for i in [0, 1] + list(range(5, 13)):
        assert L.tagi_moe_route(*_without(route, i)) == capi.ERR_INVALID_ARG
    for i, bad in ((2, 0), (3, 0), (4, 0), (4, 9), (4, -1)):
        assert L.tagi_moe_route(*_without(route, i, bad)) == capi.ERR_INVALID_ARG
    assert L.tagi_moe_route(*([one, one, 4, 1025, 2] + route[5:])) == capi.ERR_UNSUPPORTED
    assert L.tagi_moe_route(*([one, one, 4, 100, 65] + route[5:])) == capi.ERR_UNSUPPORTED
    assert L.tagi_moe_route(*([one, one, 1 << 30, 100, 4] + route[5:])) == capi.ERR_UNSUPPORTED
    size = ctypes.c_size_t(0)
    assert L.tagi_moe_route_scratch(0, 4, ctypes.byref(size)) == capi.ERR_INVALID_ARG
    assert L.tagi_moe_route_scratch(4, 1025, ctypes.byref(size)) == capi.ERR_UNSUPPORTED
    assert L.tagi_moe_route_scratch(4, 4, None) == capi.ERR_INVALID_ARG


def test_router_refuses_more_tokens_than_a_launch_holds():
    """32 tokens to a workgroup of 256 threads: the largest plan whose launch stays below 2^32
    threads has 2^29 - 32 tokens."""
    capi, L = _lib()
    route = [one, one, 0, 1, 1] + [one] * 8 + [None]
    for T in ((1 << 29) - 31, (1 << 29) - 1, 1 << 29):
        assert -(-T // 32) * 256 >= 1 << 32
        assert L.tagi_moe_route(*_without(route, 2, T)) == capi.ERR_UNSUPPORTED



def test_gated_sum_refuses():
    capi, L = _lib()
    fwd = [one] * 5 + [4, 2, 8, 16] + [one] * 2 + [None]
    for i in [0, 1, 2, 3, 4, 9, 10]:
        assert L.tagi_moe_combine_fwd(*_without(fwd, i)) == capi.ERR_INVALID_ARG
    for i in range(5, 9):
        assert L.tagi_moe_combine_fwd(*_without(fwd, i, 0)) == capi.ERR_INVALID_ARG
    bwd = [one] * 7 + [4, 2, 8, 16, 4] + [one] * 4 + [None]
    for i in list(range(7)) + list(range(12, 16)):
        assert L.tagi_moe_combine_bwd(*_without(bwd, i)) == capi.ERR_INVALID_ARG
    for i in range(7, 12):
        assert L.tagi_moe_combine_bwd(*_without(bwd, i, 0)) == capi.ERR_INVALID_ARG
    gather = [one] * 6 + [4, 2, 8, 16] + [one] * 2 + [None]
    for i in [0, 1, 2, 4, 5, 10, 11]:      # (4, 5: one of the pair alone)
        assert L.tagi_moe_gather_bwd(*_without(gather, i)) == capi.ERR_INVALID_ARG
    for i in range(6, 10):
        assert L.tagi_moe_gather_bwd(*_without(gather, i, 0)) == capi.ERR_INVALID_ARG


def test_tensor_calls_refuse():
    """Shapes, types, strides, pairs and devices."""
    import cutagi_amd.functional as F
    f = torch.ones
    i = lambda *s: torch.zeros(s, dtype=torch.int32)
    w, v = f(8), f(8)

    def no(match, call, *args, **kw):
        with pytest.raises(ValueError, match=match):
            call(*args, **kw)
    no("device tensor", F.layernorm_fwd, w, v, None, None, f(2, 8), f(2, 8))
    no("come together", F.layernorm_fwd, w, v, w, None, f(2, 8), f(2, 8))
    no("mu_w: expected shape", F.layernorm_fwd, f(7), v, None, None, f(2, 8), f(2, 8))
    no("var_a: expected a contiguous", F.layernorm_fwd, w, v, None, None, f(2, 8), f(8, 2).t())
    no("mu_a: expected a contiguous", F.layernorm_fwd, w, v, None, None, f(2, 8).half(), f(2, 8))
    no("mu_a: expected 2 dim", F.layernorm_fwd, w, v, None, None, f(8), f(8))
    no("mu_s: expected shape", F.layernorm_bwd, w, v, v, f(2, 8), None, f(3), f(2), f(2, 8), f(2, 8))
    W = f(3, 4, 8)
    no("offsets: expected shape", F.grouped_linear_fwd, W, W, None, None, f(5, 8), f(5, 8), i(3))
    no("offsets: expected a contiguous", F.grouped_linear_fwd, W, W, None, None, f(5, 8), f(5, 8), i(4).long())
    no("mu_w: expected shape", F.grouped_linear_fwd, W, W, None, None, f(5, 9), f(5, 9), i(4))
    no("var_a: expected shape", F.grouped_linear_fwd, W, W, None, None, f(5, 8), f(4, 8), i(4))
    no("mu_w: expected 3 dim", F.grouped_linear_fwd, W[0], W[0], None, None, f(5, 8), f(5, 8), i(4))
    no("rows: expected 1 dim", F.grouped_linear_fwd, W, W, None, None, f(5, 8), f(5, 8), i(4), rows=i(2, 2))
    no("come together", F.grouped_linear_fwd, W, W, f(3, 4), None, f(5, 8), f(5, 8), i(4))
    no("device tensor", F.grouped_linear_fwd, W, W, None, None, f(5, 8), f(5, 8), i(4))
    no("mu_a: expected shape", F.grouped_linear_bwd, W, W, None, f(6, 8), None, f(5, 4), f(5, 4), i(4))
    no("mu_w: expected shape|var_b: expected shape", F.grouped_linear_bwd, W, W, f(3, 5), f(5, 8), None,
       f(5, 4), f(5, 4), i(4))
    no("top_k 5", F.moe_route, f(4, 4), f(4, 4), 5)
    no("top_k 0", F.moe_route, f(4, 4), f(4, 4), 0)
    no("var_s: expected shape", F.moe_route, f(4, 4), f(4, 5), 2)
    no("slot: expected a contiguous", F.moe_combine_fwd, f(4, 2), f(4, 2), f(8, 3), f(8, 3), i(4, 2).long())
    no("expert: expected shape", F.moe_combine_bwd, f(4, 2), f(4, 2), f(8, 3), i(4, 3), i(4, 2), f(4, 3), f(4, 3), 4)
    no("come together", F.moe_gather_bwd, f(8, 3), f(8, 3), i(4, 2), None, f(4, 3), None)


def test_block_sizes_behind_an_image():
    """A Linear layer hands the image's geometry on: a block behind it has the features of its
    layers, not the image's pixels."""
    from cutagi_amd import nn
    block = lambda *tail: nn.ResNetBlock(nn.LayerBlock(nn.LayerNorm(20), nn.MixtureOfExperts(20, 24, 20, 4, 2), *tail))
    image = lambda: nn.Conv2d(1, 2, 3, padding=1, in_width=4, in_height=4)
    net = nn.Sequential(image(), nn.ReLU(), nn.Linear(32, 20), block(), nn.ReLU(), block(nn.BatchNorm2d(20), nn.ReLU()),
                        nn.Linear(20, 3))
    assert [(net.layers[i].input_size, net.layers[i].output_size) for i in (3, 5)] == [(20, 20)] * 2
    shortcut = nn.LayerBlock(nn.Linear(20, 12), nn.ReLU(), nn.Linear(12, 12))
    main = nn.LayerBlock(nn.ReLU(), nn.Linear(20, 30), nn.MixtureReLU(), nn.Linear(30, 12))
    flat = nn.Sequential(image(), nn.Linear(32, 20), nn.ResNetBlock(main, shortcut), nn.Linear(12, 3))
    assert (flat.layers[2].input_size, flat.layers[2].output_size) == (20, 12)
    # and a block of convolutions still has the image's
    conv = nn.ResNetBlock(nn.LayerBlock(nn.Conv2d(2, 2, 3, padding=1), nn.BatchNorm2d(2), nn.ReLU()))
    net = nn.Sequential(image(), nn.ReLU(), conv, nn.Linear(32, 3))
    assert (net.layers[2].input_size, net.layers[2].output_size) == (32, 32)


def test_layer_descriptions():
    """The host layers without a GPU: sizes, parameters, refusals, no CPU compute path."""
    import numpy as np
    from cutagi_amd import cutagi, nn
    cutagi.manual_seed(0)
    net = nn.Sequential(nn.LayerNorm([4, 2]), nn.MixtureOfExperts(8, 16, 4, 3, 2), nn.LayerNorm(4, bias=False))
    assert net.get_layer_stack_info().split() == ["LayerNorm()", "MixtureOfExperts(8,16,4,3,2)", "LayerNorm()"]
    sizes = {k: [len(x) for x in v] for k, v in net.state_dict().items()}
    w, b = 3 * 8 + 3 * 16 * 8 + 3 * 4 * 16, 3 + 3 * 16 + 3 * 4
    assert sizes == {"LayerNorm.0": [8] * 4, "MixtureOfExperts.1": [w, w, b, b], "LayerNorm.2": [4, 4, 0, 0]}
    mu_w, var_w = net.state_dict()["MixtureOfExperts.1"][:2]
    assert np.allclose(var_w[:24 + 384], 1 / 8) and np.allclose(var_w[24 + 384:], 1 / 16)   # He, by part
    assert net.state_dict()["LayerNorm.0"][0] == [1.0] * 8
    for make in (lambda: nn.LayerNorm(1), lambda: nn.LayerNorm([]), lambda: nn.LayerNorm([4, 0]),
                 lambda: nn.MixtureOfExperts(8, 16, 4, 3, 4), lambda: nn.MixtureOfExperts(8, 16, 4, 3, 0),
                 lambda: nn.MixtureOfExperts(0, 16, 4, 3, 2), lambda: nn.MixtureOfExperts(8, 16, 4, 2000, 2),
                 lambda: nn.MixtureOfExperts(8, 16, 4, 3, 2, "tanh")):
        with pytest.raises(RuntimeError):
            make()
    with pytest.raises(RuntimeError, match="GPU only"):
        net.forward(np.zeros((2, 8), np.float32))
