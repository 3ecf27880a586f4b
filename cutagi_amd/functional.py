"""Tensor-level calls into the C ABI.

torch is plumbing here: it owns device memory and the current stream; every
computation is one C-ABI call on raw pointers. Shapes follow the reference:
weights [N, K], activations [B, K], conv weights [fo, fi*k*k], conv activations
flattened NCHW.
"""
import collections

import torch

from . import capi


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _chk(*tensors):
    for t in tensors:
        if t is None:
            continue
        if not (t.is_cuda and t.is_contiguous() and t.dtype in (torch.float32, torch.int32)):
            raise ValueError("expected contiguous fp32/int32 device tensors")


def linear_fwd(mu_w, var_w, mu_b, var_b, mu_a, var_a, out=None):
    _chk(mu_w, var_w, mu_b, var_b, mu_a, var_a)
    N, K = mu_w.shape
    B = mu_a.shape[0]
    if mu_a.shape[1] != K:
        raise ValueError("Input size mismatch: %d vs %d" % (K, mu_a.shape[1]))
    mu_z, var_z = out if out is not None else (torch.empty((B, N), device=mu_w.device),
                                                torch.empty((B, N), device=mu_w.device))
    bias = mu_b is not None
    capi.check(capi.lib.tagi_linear_fwd(capi.ptr(mu_w), capi.ptr(var_w), capi.ptr(mu_b),
                                        capi.ptr(var_b), capi.ptr(mu_a), capi.ptr(var_a), K, N, B,
                                        int(bias), capi.ptr(mu_z), capi.ptr(var_z), _stream()))
    return mu_z, var_z


ACTIVATIONS = {"relu": 1, "mixture_relu": 2}


def linear_fwd_act(mu_w, var_w, mu_b, var_b, mu_a, var_a, activation):
    """Linear forward with the following activation ("relu" / "mixture_relu") applied
    in the kernel's epilogue: returns the activation's (mu_a, var_a, jcb)."""
    _chk(mu_w, var_w, mu_b, var_b, mu_a, var_a)
    N, K = mu_w.shape
    B = mu_a.shape[0]
    out = [torch.empty((B, N), device=mu_w.device) for _ in range(3)]
    capi.check(capi.lib.tagi_linear_fwd_act(capi.ptr(mu_w), capi.ptr(var_w), capi.ptr(mu_b),
                                            capi.ptr(var_b), capi.ptr(mu_a), capi.ptr(var_a), K, N,
                                            B, int(mu_b is not None), ACTIVATIONS[activation],
                                            capi.ptr(out[0]), capi.ptr(out[1]), capi.ptr(out[2]),
                                            _stream()))
    return tuple(out)


def linear_bwd_dz(mu_w, jcb, delta_mu, delta_var, out=None):
    _chk(mu_w, jcb, delta_mu, delta_var)
    N, K = mu_w.shape
    B = delta_mu.shape[0]
    om, ov = out if out is not None else (torch.empty((B, K), device=mu_w.device),
                                          torch.empty((B, K), device=mu_w.device))
    capi.check(capi.lib.tagi_linear_bwd_dz(capi.ptr(mu_w), capi.ptr(jcb), capi.ptr(delta_mu),
                                           capi.ptr(delta_var), K, N, B, capi.ptr(om),
                                           capi.ptr(ov), _stream()))
    return om, ov


def linear_bwd_dw(var_w, mu_a, delta_mu, delta_var, out=None):
    _chk(var_w, mu_a, delta_mu, delta_var)
    N, K = var_w.shape
    B = delta_mu.shape[0]
    om, ov = out if out is not None else (torch.empty((N, K), device=var_w.device),
                                          torch.empty((N, K), device=var_w.device))
    capi.check(capi.lib.tagi_linear_bwd_dw(capi.ptr(var_w), capi.ptr(mu_a), capi.ptr(delta_mu),
                                           capi.ptr(delta_var), K, N, B, capi.ptr(om),
                                           capi.ptr(ov), _stream()))
    return om, ov


def linear_bwd_db(var_b, delta_mu, delta_var, out=None):
    _chk(var_b, delta_mu, delta_var)
    B, N = delta_mu.shape
    om, ov = out if out is not None else (torch.empty(N, device=var_b.device),
                                          torch.empty(N, device=var_b.device))
    capi.check(capi.lib.tagi_linear_bwd_db(capi.ptr(var_b), capi.ptr(delta_mu),
                                           capi.ptr(delta_var), N, B, capi.ptr(om), capi.ptr(ov),
                                           _stream()))
    return om, ov


def linear_bwd(mu_w, var_w, var_b, mu_a, jcb, delta_mu, delta_var, state_update=True,
               param_update=True, out=None):
    """All of LinearCuda::backward in one call. Returns (dz_mu, dz_var, dw_mu,
    dw_var, db_mu, db_var); entries not asked for are None."""
    _chk(mu_w, var_w, var_b, mu_a, jcb, delta_mu, delta_var)
    N, K = mu_w.shape
    B = delta_mu.shape[0]
    dev = mu_w.device
    bias = var_b is not None
    if out is None:
        out = [None] * 6
        if state_update:
            out[0], out[1] = torch.empty((B, K), device=dev), torch.empty((B, K), device=dev)
        if param_update:
            out[2], out[3] = torch.empty((N, K), device=dev), torch.empty((N, K), device=dev)
            if bias:
                out[4], out[5] = torch.empty(N, device=dev), torch.empty(N, device=dev)
    capi.check(capi.lib.tagi_linear_bwd(
        capi.ptr(mu_w), capi.ptr(var_w), capi.ptr(var_b), capi.ptr(mu_a), capi.ptr(jcb),
        capi.ptr(delta_mu), capi.ptr(delta_var), K, N, B, int(bias), int(state_update),
        int(param_update), *[capi.ptr(t) for t in out], _stream()))
    return tuple(out)


def conv2d_fwd(mu_w, var_w, mu_b, var_b, mu_a, var_a, aidx, woho, fo, wihi, fi, ki, B):
    _chk(mu_w, var_w, mu_b, var_b, mu_a, var_a, aidx)
    mu_z = torch.empty(B * fo * woho, device=mu_w.device)
    var_z = torch.empty(B * fo * woho, device=mu_w.device)
    bias = mu_b is not None
    capi.check(capi.lib.tagi_conv2d_fwd(capi.ptr(mu_w), capi.ptr(var_w), capi.ptr(mu_b),
                                        capi.ptr(var_b), capi.ptr(mu_a), capi.ptr(var_a),
                                        capi.ptr(aidx), woho, fo, wihi, fi, ki, B, int(bias),
                                        capi.ptr(mu_z), capi.ptr(var_z), _stream()))
    return mu_z, var_z


def conv2d_fwd_act(mu_w, var_w, mu_b, var_b, mu_a, var_a, aidx, woho, fo, wihi, fi, ki, B,
                   activation):
    """Conv2d forward with the following activation applied in the kernel's epilogue:
    returns the activation's (mu_a, var_a, jcb), each [B][fo][woho] flattened."""
    _chk(mu_w, var_w, mu_b, var_b, mu_a, var_a, aidx)
    out = [torch.empty(B * fo * woho, device=mu_w.device) for _ in range(3)]
    capi.check(capi.lib.tagi_conv2d_fwd_act(capi.ptr(mu_w), capi.ptr(var_w), capi.ptr(mu_b),
                                            capi.ptr(var_b), capi.ptr(mu_a), capi.ptr(var_a),
                                            capi.ptr(aidx), woho, fo, wihi, fi, ki, B,
                                            int(mu_b is not None), ACTIVATIONS[activation],
                                            capi.ptr(out[0]), capi.ptr(out[1]), capi.ptr(out[2]),
                                            _stream()))
    return tuple(out)


def conv2d_bwd_dz(mu_w, jcb, delta_mu, delta_var, zw_idx, zud_idx, woho, fo, wihi, fi, ki, nr, B):
    _chk(mu_w, jcb, delta_mu, delta_var, zw_idx, zud_idx)
    om = torch.empty(B * fi * wihi, device=mu_w.device)
    ov = torch.empty(B * fi * wihi, device=mu_w.device)
    capi.check(capi.lib.tagi_conv2d_bwd_dz(capi.ptr(mu_w), capi.ptr(jcb), capi.ptr(delta_mu),
                                           capi.ptr(delta_var), capi.ptr(zw_idx),
                                           capi.ptr(zud_idx), woho, fo, wihi, fi, ki, nr, B,
                                           capi.ptr(om), capi.ptr(ov), _stream()))
    return om, ov


def conv2d_bwd_dw(var_w, var_b, mu_a, delta_mu, delta_var, aidx, B, fo, woho, wihi, fi, ki):
    _chk(var_w, var_b, mu_a, delta_mu, delta_var, aidx)
    nw = ki * ki * fi * fo
    dev = var_w.device
    om, ov = torch.empty(nw, device=dev), torch.empty(nw, device=dev)
    bias = var_b is not None
    bm = torch.empty(fo, device=dev) if bias else None
    bv = torch.empty(fo, device=dev) if bias else None
    capi.check(capi.lib.tagi_conv2d_bwd_dw(capi.ptr(var_w), capi.ptr(var_b), capi.ptr(mu_a),
                                           capi.ptr(delta_mu), capi.ptr(delta_var),
                                           capi.ptr(aidx), B, fo, woho, wihi, fi, ki, int(bias),
                                           capi.ptr(om), capi.ptr(ov), capi.ptr(bm), capi.ptr(bv),
                                           _stream()))
    return om, ov, bm, bv


def conv2d_bwd(mu_w, var_w, var_b, mu_a, jcb, delta_mu, delta_var, aidx, zw_idx, zud_idx, B, fo,
               woho, wihi, fi, ki, nr, state_update=True, param_update=True, res_mu=None,
               res_var=None, res_mode=0):
    """Both backward contractions in one call: (delta_mu_z, delta_var_z, delta_mu_w,
    delta_var_w, delta_mu_b, delta_var_b), None where a part is switched off."""
    _chk(mu_w, var_w, var_b, mu_a, jcb, delta_mu, delta_var, aidx, zw_idx, zud_idx, res_mu, res_var)
    dev = mu_w.device
    nw = ki * ki * fi * fo
    bias = var_b is not None
    zm = torch.empty(B * fi * wihi, device=dev) if state_update else None
    zv = torch.empty(B * fi * wihi, device=dev) if state_update else None
    wm = torch.empty(nw, device=dev) if param_update else None
    wv = torch.empty(nw, device=dev) if param_update else None
    bm = torch.empty(fo, device=dev) if bias and param_update else None
    bv = torch.empty(fo, device=dev) if bias and param_update else None
    capi.check(capi.lib.tagi_conv2d_bwd(
        capi.ptr(mu_w), capi.ptr(var_w), capi.ptr(var_b), capi.ptr(mu_a), capi.ptr(jcb),
        capi.ptr(delta_mu), capi.ptr(delta_var), capi.ptr(aidx), capi.ptr(zw_idx), capi.ptr(zud_idx),
        B, fo, woho, wihi, fi, ki, nr, int(bias), int(state_update), int(param_update),
        capi.ptr(res_mu), capi.ptr(res_var), res_mode, capi.ptr(zm), capi.ptr(zv), capi.ptr(wm),
        capi.ptr(wv), capi.ptr(bm), capi.ptr(bv), _stream()))
    return zm, zv, wm, wv, bm, bv


def store_states(mu_a, jcb, n_in, bwd_mu_a, bwd_jcb, out_jcb, n_out):
    capi.check(capi.lib.tagi_store_states(capi.ptr(mu_a), capi.ptr(jcb), n_in, capi.ptr(bwd_mu_a),
                                          capi.ptr(bwd_jcb), capi.ptr(out_jcb), n_out, _stream()))


def param_update(delta_mu, delta_var, cap_factor, mu, var, neg_var_count=None):
    """In place on mu/var. neg_var_count: int32 device tensor of one element."""
    _chk(delta_mu, delta_var, mu, var, neg_var_count)
    capi.check(capi.lib.tagi_param_update(capi.ptr(delta_mu), capi.ptr(delta_var), cap_factor,
                                          mu.numel(), capi.ptr(mu), capi.ptr(var),
                                          capi.ptr(neg_var_count), _stream()))



def layer_update(delta_mu_w, delta_var_w, mu_w, var_w, delta_mu_b, delta_var_b, mu_b, var_b,
                 cap_factor, neg_var_count=None, slot=0):
    """Weights and biases of a layer in one launch, in place. Bias tensors may be
    None. neg_var_count: int32 device tensor of two elements (counts go to [slot],
    [1 - slot] is zeroed)."""
    _chk(delta_mu_w, delta_var_w, mu_w, var_w, delta_mu_b, delta_var_b, mu_b, var_b, neg_var_count)
    nb = 0 if mu_b is None else mu_b.numel()
    capi.check(capi.lib.tagi_layer_update(
        capi.ptr(delta_mu_w), capi.ptr(delta_var_w), mu_w.numel(), capi.ptr(mu_w), capi.ptr(var_w),
        capi.ptr(delta_mu_b), capi.ptr(delta_var_b), nb, capi.ptr(mu_b), capi.ptr(var_b),
        cap_factor, capi.ptr(neg_var_count), int(slot), _stream()))

def out_update_dense(mu_a, var_a, jcb, obs, var_obs, delta_mu, delta_var):
    _chk(mu_a, var_a, jcb, obs, var_obs, delta_mu, delta_var)
    capi.check(capi.lib.tagi_out_update_dense(capi.ptr(mu_a), capi.ptr(var_a), capi.ptr(jcb),
                                              capi.ptr(obs), capi.ptr(var_obs), obs.numel(),
                                              capi.ptr(delta_mu), capi.ptr(delta_var), _stream()))


def out_update_heteros(mu_a, var_a, jcb, obs, delta_mu, delta_var):
    """obs.numel() observations against 2 * obs.numel() output units."""
    _chk(mu_a, var_a, jcb, obs, delta_mu, delta_var)
    capi.check(capi.lib.tagi_out_update_heteros(capi.ptr(mu_a), capi.ptr(var_a), capi.ptr(jcb),
                                                capi.ptr(obs), obs.numel(), capi.ptr(delta_mu),
                                                capi.ptr(delta_var), _stream()))


def out_update_indexed(mu_a, var_a, jcb, obs, var_obs, selected_idx, n_obs, n_enc, delta_mu,
                       delta_var):
    _chk(mu_a, var_a, jcb, obs, var_obs, selected_idx, delta_mu, delta_var)
    capi.check(capi.lib.tagi_out_update_indexed(capi.ptr(mu_a), capi.ptr(var_a), capi.ptr(jcb),
                                                capi.ptr(obs), capi.ptr(var_obs),
                                                capi.ptr(selected_idx), n_obs, n_enc, obs.numel(),
                                                capi.ptr(delta_mu), capi.ptr(delta_var),
                                                _stream()))


def relu_fwd(mu_z, var_z, mu_a=None, jcb=None, var_a=None):
    _chk(mu_z, var_z, mu_a, jcb, var_a)
    mu_a = torch.empty_like(mu_z) if mu_a is None else mu_a
    jcb = torch.empty_like(mu_z) if jcb is None else jcb
    var_a = torch.empty_like(mu_z) if var_a is None else var_a
    capi.check(capi.lib.tagi_relu_fwd(capi.ptr(mu_z), capi.ptr(var_z), mu_z.numel(),
                                      capi.ptr(mu_a), capi.ptr(jcb), capi.ptr(var_a), _stream()))
    return mu_a, var_a, jcb


def mixture_relu_fwd(mu_z, var_z, mu_a=None, jcb=None, var_a=None):
    _chk(mu_z, var_z, mu_a, jcb, var_a)
    mu_a = torch.empty_like(mu_z) if mu_a is None else mu_a
    jcb = torch.empty_like(mu_z) if jcb is None else jcb
    var_a = torch.empty_like(mu_z) if var_a is None else var_a
    capi.check(capi.lib.tagi_mixture_relu_fwd(capi.ptr(mu_z), capi.ptr(var_z), mu_z.numel(),
                                              capi.ptr(mu_a), capi.ptr(jcb), capi.ptr(var_a),
                                              _stream()))
    return mu_a, var_a, jcb


def batchnorm2d_stats(mu_a, var_a, wihi, fi, B, momentum, mu_ra, var_ra):
    """Batch statistics (returned) and the running averages (updated in place)."""
    _chk(mu_a, var_a, mu_ra, var_ra)
    mu_s, var_s = torch.empty(fi, device=mu_a.device), torch.empty(fi, device=mu_a.device)
    capi.check(capi.lib.tagi_batchnorm2d_stats(capi.ptr(mu_a), capi.ptr(var_a), wihi, fi, B,
                                               momentum, capi.ptr(mu_s), capi.ptr(var_s),
                                               capi.ptr(mu_ra), capi.ptr(var_ra), _stream()))
    return mu_s, var_s


def batchnorm2d_fwd(mu_w, var_w, mu_b, var_b, mu_a, var_a, mu_norm, var_norm, eps, wihi, fi, B):
    _chk(mu_w, var_w, mu_b, var_b, mu_a, var_a, mu_norm, var_norm)
    mu_z, var_z = torch.empty_like(mu_a), torch.empty_like(mu_a)
    capi.check(capi.lib.tagi_batchnorm2d_fwd(capi.ptr(mu_w), capi.ptr(var_w), capi.ptr(mu_b),
                                             capi.ptr(var_b), capi.ptr(mu_a), capi.ptr(var_a),
                                             capi.ptr(mu_norm), capi.ptr(var_norm),
                                             int(mu_b is not None), eps, wihi, fi, B,
                                             capi.ptr(mu_z), capi.ptr(var_z), _stream()))
    return mu_z, var_z


def batchnorm2d_bwd(mu_w, var_w, var_b, mu_a, jcb, mu_norm, var_norm, delta_mu, delta_var, eps,
                    wihi, fi, B, state_update=True, param_update=True):
    """Returns (dz_mu, dz_var, dw_mu, dw_var, db_mu, db_var); entries not asked for are None."""
    _chk(mu_w, var_w, var_b, mu_a, jcb, mu_norm, var_norm, delta_mu, delta_var)
    dev = mu_w.device
    bias = var_b is not None
    out = [None] * 6
    if state_update:
        out[0], out[1] = torch.empty_like(delta_mu), torch.empty_like(delta_mu)
    if param_update:
        out[2], out[3] = torch.empty(fi, device=dev), torch.empty(fi, device=dev)
        if bias:
            out[4], out[5] = torch.empty(fi, device=dev), torch.empty(fi, device=dev)
    capi.check(capi.lib.tagi_batchnorm2d_bwd(
        capi.ptr(mu_w), capi.ptr(var_w), capi.ptr(var_b), capi.ptr(mu_a), capi.ptr(jcb),
        capi.ptr(mu_norm), capi.ptr(var_norm), capi.ptr(delta_mu), capi.ptr(delta_var), eps, wihi,
        fi, B, int(bias), int(state_update), int(param_update), *[capi.ptr(t) for t in out],
        _stream()))
    return tuple(out)


def avgpool2d_fwd(mu_a, var_a, pool_idx, woho, wihi, ki, n_out):
    _chk(mu_a, var_a, pool_idx)
    mu_z, var_z = torch.empty(n_out, device=mu_a.device), torch.empty(n_out, device=mu_a.device)
    capi.check(capi.lib.tagi_avgpool2d_fwd(capi.ptr(mu_a), capi.ptr(var_a), capi.ptr(pool_idx),
                                           woho, wihi, ki, n_out, capi.ptr(mu_z), capi.ptr(var_z),
                                           _stream()))
    return mu_z, var_z


def avgpool2d_bwd_dz(jcb, delta_mu, delta_var, z_ud_idx, woho, wihi, ki, nr, wo, overlap):
    _chk(jcb, delta_mu, delta_var, z_ud_idx)
    om, ov = torch.empty_like(jcb), torch.empty_like(jcb)
    capi.check(capi.lib.tagi_avgpool2d_bwd_dz(capi.ptr(jcb), capi.ptr(delta_mu),
                                              capi.ptr(delta_var), capi.ptr(z_ud_idx), woho, wihi,
                                              ki, nr, wo, jcb.numel(), int(overlap), capi.ptr(om),
                                              capi.ptr(ov), _stream()))
    return om, ov


def add_shortcut(mu_s, var_s, mu_a, var_a):
    """In place on mu_a/var_a."""
    _chk(mu_s, var_s, mu_a, var_a)
    capi.check(capi.lib.tagi_add_shortcut(capi.ptr(mu_s), capi.ptr(var_s), mu_a.numel(),
                                          capi.ptr(mu_a), capi.ptr(var_a), _stream()))


def add_shortcut_delta(mu_s, var_s, jcb_s, mu_a, var_a):
    """In place on mu_a/var_a."""
    _chk(mu_s, var_s, jcb_s, mu_a, var_a)
    capi.check(capi.lib.tagi_add_shortcut_delta(capi.ptr(mu_s), capi.ptr(var_s), capi.ptr(jcb_s),
                                                mu_a.numel(), capi.ptr(mu_a), capi.ptr(var_a),
                                                _stream()))


# ---- layer norm, grouped Linear layers, mixture of experts ---------------------------------
# Calls for single tokens are bound by the host, so these keep to a few allocations each and
# name what is wrong with an argument only once something is.

_F, _I = torch.float32, torch.int32


def _fits(device, dtype, shape, *tensors):
    """Whether every tensor (None: absent) is a contiguous one of this device, type and shape."""
    for t in tensors:
        if t is not None and (t.dtype is not dtype or t.shape != shape or not t.is_contiguous()
                              or t.get_device() != device):
            return False
    return True


def _explain(**named):
    """Raises for the first argument, name -> (tensor or None, shape, dtype), that is not a
    contiguous tensor of that shape and type on the current device."""
    present = [(name, t, shape, dtype) for name, (t, shape, dtype) in named.items() if t is not None]
    for name, t, shape, dtype in present:
        if t.dtype != dtype or not t.is_contiguous():
            raise ValueError("%s: expected a contiguous %s tensor" % (name, dtype))
        if tuple(t.shape) != tuple(shape):
            raise ValueError("%s: expected shape %s, got %s" % (name, tuple(shape), tuple(t.shape)))
    for name, t, _, _ in present:
        if not t.is_cuda:
            raise ValueError("%s: expected a device tensor" % name)
        if t.device.index != torch.cuda.current_device():
            raise ValueError("%s is on %s, the current device is cuda:%d"
                             % (name, t.device, torch.cuda.current_device()))
    raise ValueError("arguments on more than one device")


def _device(t):
    """Index of the current device for calls that start from tensor t (-2 for a host tensor:
    nothing fits it)."""
    return torch._C._cuda_getDevice() if t.is_cuda else -2


def _raw_stream(device):
    return torch._C._cuda_getCurrentRawStream(device)


def _at(t):
    return None if t is None else t.data_ptr()


def _pair(a, b, names):
    if (a is None) != (b is None):
        raise ValueError("%s and %s come together" % names)


def _dims(name, t, n):
    """The n sizes of a tensor argument."""
    if t.dim() != n:
        raise ValueError("%s: expected %d dimensions, got %s" % (name, n, tuple(t.shape)))
    return t.shape


def _new(like, count, *shape):
    """`count` new fp32 tensors of a shape, from one allocation."""
    return like.new_empty((count,) + shape, dtype=_F).unbind(0)


def layernorm_fwd(mu_w, var_w, mu_b, var_b, mu_a, var_a, eps=1e-5):
    """Layer norm over the last dimension of mu_a / var_a [B, n]: (mu_z, var_z, mu_s, var_s),
    mu_s / var_s [B] the statistics of the rows. mu_b / var_b may be None."""
    _pair(mu_b, var_b, ("mu_b", "var_b"))
    B, n = _dims("mu_a", mu_a, 2)
    dev = _device(mu_a)
    if not (_fits(dev, _F, (B, n), mu_a, var_a) and _fits(dev, _F, (n,), mu_w, var_w, mu_b, var_b)):
        _explain(mu_a=(mu_a, (B, n), _F), var_a=(var_a, (B, n), _F), mu_w=(mu_w, (n,), _F),
                 var_w=(var_w, (n,), _F), mu_b=(mu_b, (n,), _F), var_b=(var_b, (n,), _F))
    mu_z, var_z = _new(mu_a, 2, B, n)
    mu_s, var_s = _new(mu_a, 2, B)
    capi.check(capi.lib.tagi_layernorm_fwd(
        mu_w.data_ptr(), var_w.data_ptr(), _at(mu_b), _at(var_b), mu_a.data_ptr(),
        var_a.data_ptr(), int(mu_b is not None), eps, n, B, mu_s.data_ptr(), var_s.data_ptr(),
        mu_z.data_ptr(), var_z.data_ptr(), _raw_stream(dev)))
    return mu_z, var_z, mu_s, var_s


def layernorm_bwd(mu_w, var_w, var_b, mu_a, jcb, mu_s, var_s, delta_mu, delta_var, eps=1e-5,
                  state_update=True, param_update=True):
    """Returns (dz_mu, dz_var, dw_mu, dw_var, db_mu, db_var); entries not asked for are None.
    jcb may be None (one everywhere)."""
    B, n = _dims("delta_mu", delta_mu, 2)
    dev = _device(delta_mu)
    if not (_fits(dev, _F, (B, n), delta_mu, delta_var, mu_a, jcb) and
            _fits(dev, _F, (n,), mu_w, var_w, var_b) and _fits(dev, _F, (B,), mu_s, var_s)):
        _explain(delta_mu=(delta_mu, (B, n), _F), delta_var=(delta_var, (B, n), _F),
                 mu_w=(mu_w, (n,), _F), var_w=(var_w, (n,), _F), var_b=(var_b, (n,), _F),
                 mu_a=(mu_a, (B, n), _F), jcb=(jcb, (B, n), _F), mu_s=(mu_s, (B,), _F),
                 var_s=(var_s, (B,), _F))
    out, scratch = [None] * 6, None
    if state_update:
        out[:2] = _new(delta_mu, 2, B, n)
    if param_update:
        count = 2 if var_b is None else 4
        out[2:2 + count] = _new(delta_mu, count, n)
        size = capi.layernorm_bwd_scratch(n, B)
        scratch = delta_mu.new_empty(size, dtype=torch.uint8) if size else None
    capi.check(capi.lib.tagi_layernorm_bwd(
        mu_w.data_ptr(), var_w.data_ptr(), _at(var_b), mu_a.data_ptr(), _at(jcb), mu_s.data_ptr(),
        var_s.data_ptr(), delta_mu.data_ptr(), delta_var.data_ptr(), eps, n, B,
        int(var_b is not None), int(state_update), int(param_update), _at(scratch),
        *[_at(t) for t in out], _raw_stream(dev)))
    return tuple(out)


def grouped_linear_fwd(mu_w, var_w, mu_b, var_b, mu_a, var_a, offsets, rows=None, out=None):
    """Linear layers [E, N, K], rows grouped by expert: rows offsets[e] .. offsets[e+1] meet
    the weights of expert e (offsets: int32 [E+1]). rows (int32 [R]): row r is row rows[r] of
    mu_a / var_a; without it mu_a / var_a [R, K] hold the rows in order. Returns (mu_z, var_z)
    [R, N]; rows from offsets[E] on are left as `out` held them (unset without `out`).
    Which kernels a call runs on depends on all of its sizes; some take fp32 numbers apart into
    three bf16 parts, and there (here and in grouped_linear_bwd) an infinity may come out as
    NaN and numbers below 3e-33 count with less than fp32's precision."""
    return _grouped_fwd(mu_w, var_w, mu_b, var_b, mu_a, var_a, offsets, rows, None, out)


def grouped_linear_fwd_act(mu_w, var_w, mu_b, var_b, mu_a, var_a, offsets, activation, rows=None,
                           out=None):
    """grouped_linear_fwd with the following activation ("relu" / "mixture_relu") applied in
    the kernel's epilogue: returns the activation's (mu_a, var_a, jcb), each [R, N]."""
    return _grouped_fwd(mu_w, var_w, mu_b, var_b, mu_a, var_a, offsets, rows, ACTIVATIONS[activation],
                        out)


def _grouped_scratch(like, K, N, E, R):
    size = capi.grouped_linear_scratch(K, N, E, R)
    return like.new_empty(size, dtype=torch.uint8) if size else None


def _grouped_fwd(mu_w, var_w, mu_b, var_b, mu_a, var_a, offsets, rows, activation, out):
    _pair(mu_b, var_b, ("mu_b", "var_b"))
    T, K = _dims("mu_a", mu_a, 2)
    R = T if rows is None else _dims("rows", rows, 1)[0]
    E, N, _ = _dims("mu_w", mu_w, 3)
    dev = _device(mu_a)
    count = 2 if activation is None else 3
    if out is not None and len(out) != count:
        raise ValueError("out: expected %d tensors" % count)
    if not (_fits(dev, _F, (E, N, K), mu_w, var_w) and _fits(dev, _F, (E, N), mu_b, var_b) and
            _fits(dev, _F, (T, K), mu_a, var_a) and _fits(dev, _I, (E + 1,), offsets) and
            _fits(dev, _I, (R,), rows) and _fits(dev, _F, (R, N), *(out or ()))):
        _explain(mu_w=(mu_w, (E, N, K), _F), var_w=(var_w, (E, N, K), _F), mu_b=(mu_b, (E, N), _F),
                 var_b=(var_b, (E, N), _F), mu_a=(mu_a, (T, K), _F), var_a=(var_a, (T, K), _F),
                 offsets=(offsets, (E + 1,), _I), rows=(rows, (R,), _I),
                 **{"out[%d]" % i: (t, (R, N), _F) for i, t in enumerate(out or ())})
    if out is None:
        out = _new(mu_w, count, R, N)
    args = (mu_w.data_ptr(), var_w.data_ptr(), _at(mu_b), _at(var_b), mu_a.data_ptr(),
            var_a.data_ptr(), offsets.data_ptr(), _at(rows), K, N, E, R, T, int(mu_b is not None))
    scratch = _grouped_scratch(mu_w, K, N, E, R)
    outs = [_at(scratch)] + [t.data_ptr() for t in out]
    if activation is None:
        capi.check(capi.lib.tagi_grouped_linear_fwd(*args, *outs, _raw_stream(dev)))
    else:
        capi.check(capi.lib.tagi_grouped_linear_fwd_act(*args, activation, *outs, _raw_stream(dev)))
    return tuple(out)


def grouped_linear_bwd(mu_w, var_w, var_b, mu_a, jcb, delta_mu, delta_var, offsets, rows=None,
                       state_update=True, param_update=True, out=None):
    """All of the backward pass: (dz_mu, dz_var [R, K], dw_mu, dw_var [E, N, K], db_mu, db_var
    [E, N]); entries not asked for are None. dz is per row, also with `rows` (see
    moe_gather_bwd); jcb [R, K] may be None (one everywhere). Rows from offsets[E] on are left
    as out[0] and out[1] held them (unset without `out`)."""
    R, _ = _dims("delta_mu", delta_mu, 2)
    T, K = _dims("mu_a", mu_a, 2)
    E, N, _ = _dims("mu_w", mu_w, 3)
    dev, bias = _device(delta_mu), var_b is not None
    held = T if rows is not None else R
    shapes = [(R, K)] * 2 + [(E, N, K)] * 2 + [(E, N)] * 2
    wanted = [state_update] * 2 + [param_update] * 2 + [param_update and bias] * 2
    if out is not None and (len(out) != 6 or any(w and t is None for w, t in zip(wanted, out))):
        raise ValueError("out: six entries, None only where nothing is asked for")
    if not (_fits(dev, _F, (E, N, K), mu_w, var_w) and _fits(dev, _F, (E, N), var_b) and
            _fits(dev, _F, (held, K), mu_a) and _fits(dev, _I, (E + 1,), offsets) and
            _fits(dev, _I, (R,), rows) and _fits(dev, _F, (R, N), delta_mu, delta_var) and
            _fits(dev, _F, (R, K), jcb) and
            all(_fits(dev, _F, s, t) for s, t in zip(shapes, out or ()))):
        _explain(mu_w=(mu_w, (E, N, K), _F), var_w=(var_w, (E, N, K), _F), var_b=(var_b, (E, N), _F),
                 mu_a=(mu_a, (held, K), _F), offsets=(offsets, (E + 1,), _I), rows=(rows, (R,), _I),
                 delta_mu=(delta_mu, (R, N), _F), delta_var=(delta_var, (R, N), _F),
                 jcb=(jcb, (R, K), _F),
                 **{"out[%d]" % i: (t, s, _F) for i, (t, s) in enumerate(zip(out or (), shapes))})
    if out is None:
        out = [None] * 6
        for i in (0, 2, 4):
            if wanted[i]:
                out[i:i + 2] = _new(delta_mu, 2, *shapes[i])
    scratch = _grouped_scratch(mu_w, K, N, E, R)
    capi.check(capi.lib.tagi_grouped_linear_bwd(
        mu_w.data_ptr(), var_w.data_ptr(), _at(var_b), mu_a.data_ptr(), _at(jcb),
        delta_mu.data_ptr(), delta_var.data_ptr(), offsets.data_ptr(), _at(rows), K, N, E, R, T,
        int(bias), int(state_update), int(param_update), _at(scratch), *[_at(t) for t in out],
        _raw_stream(dev)))
    return tuple(t if w else None for w, t in zip(wanted, out))


MoeRoutes = collections.namedtuple("MoeRoutes", "expert mu_g var_g jcb_g offsets token slot")


def moe_route(mu_s, var_s, top_k):
    """The router's choice from its scores [T, E]: the top_k experts of the largest means
    (ties: lowest index; -inf and NaN are never chosen), their softmax gates, and the rows
    sorted by expert and then by token. Returns MoeRoutes: expert, mu_g, var_g, jcb_g and slot
    (the row of the choice) [T, top_k], offsets [E+1], token (of every row) [T*top_k]; -1 in
    expert, slot and token where there is nothing."""
    T, E = _dims("mu_s", mu_s, 2)
    if not 1 <= top_k <= E:
        raise ValueError("top_k %d: expected 1 to %d" % (top_k, E))
    dev = _device(mu_s)
    if not _fits(dev, _F, (T, E), mu_s, var_s):
        _explain(mu_s=(mu_s, (T, E), _F), var_s=(var_s, (T, E), _F))
    size = capi.moe_route_scratch(T, E)
    scratch = mu_s.new_empty(size, dtype=torch.uint8) if size else None
    mu_g, var_g, jcb_g = _new(mu_s, 3, T, top_k)
    # expert, slot, token, then offsets
    n = T * top_k
    whole = mu_s.new_empty(3 * n + E + 1, dtype=_I)
    expert, slot, token, offsets = whole.split((n, n, n, E + 1))
    expert, slot = expert.view(T, top_k), slot.view(T, top_k)
    at = whole.data_ptr()
    capi.check(capi.lib.tagi_moe_route(
        mu_s.data_ptr(), var_s.data_ptr(), T, E, top_k, _at(scratch), at, mu_g.data_ptr(),
        var_g.data_ptr(), jcb_g.data_ptr(), at + 12 * n, at + 8 * n, at + 4 * n, _raw_stream(dev)))
    return MoeRoutes(expert, mu_g, var_g, jcb_g, offsets, token, slot)


def moe_combine_fwd(mu_g, var_g, mu_y, var_y, slot):
    """The gated sum of the experts' outputs mu_y / var_y [R, N]: (mu_z, var_z) [T, N]. A
    choice whose slot is no row adds nothing."""
    T, k = _dims("mu_g", mu_g, 2)
    R, N = _dims("mu_y", mu_y, 2)
    dev = _device(mu_y)
    if not (_fits(dev, _F, (T, k), mu_g, var_g) and _fits(dev, _I, (T, k), slot) and
            _fits(dev, _F, (R, N), mu_y, var_y)):
        _explain(mu_g=(mu_g, (T, k), _F), var_g=(var_g, (T, k), _F), slot=(slot, (T, k), _I),
                 mu_y=(mu_y, (R, N), _F), var_y=(var_y, (R, N), _F))
    mu_z, var_z = _new(mu_y, 2, T, N)
    capi.check(capi.lib.tagi_moe_combine_fwd(
        mu_g.data_ptr(), var_g.data_ptr(), mu_y.data_ptr(), var_y.data_ptr(), slot.data_ptr(), T, k,
        R, N, mu_z.data_ptr(), var_z.data_ptr(), _raw_stream(dev)))
    return mu_z, var_z


def moe_combine_bwd(mu_g, jcb_g, mu_y, expert, slot, delta_mu, delta_var, num_experts, out=None):
    """Backward of moe_combine_fwd: (delta_mu_y, delta_var_y [R, N], delta_mu_s, delta_var_s
    [T, num_experts]), the innovations of the experts' outputs and of the router's scores.
    Rows that no choice names are left as `out` (two tensors [R, N]) held them (unset without
    `out`)."""
    T, k = _dims("mu_g", mu_g, 2)
    R, N = _dims("mu_y", mu_y, 2)
    dev = _device(mu_y)
    if out is not None and len(out) != 2:
        raise ValueError("out: expected 2 tensors")
    if not (_fits(dev, _F, (T, k), mu_g, jcb_g) and _fits(dev, _I, (T, k), expert, slot) and
            _fits(dev, _F, (R, N), mu_y, *(out or ())) and _fits(dev, _F, (T, N), delta_mu, delta_var)):
        _explain(mu_g=(mu_g, (T, k), _F), jcb_g=(jcb_g, (T, k), _F), expert=(expert, (T, k), _I),
                 slot=(slot, (T, k), _I), mu_y=(mu_y, (R, N), _F), delta_mu=(delta_mu, (T, N), _F),
                 delta_var=(delta_var, (T, N), _F),
                 **{"out[%d]" % i: (t, (R, N), _F) for i, t in enumerate(out or ())})
    dmu_y, dvar_y = out if out is not None else _new(mu_y, 2, R, N)
    dmu_s, dvar_s = _new(mu_y, 2, T, num_experts)
    capi.check(capi.lib.tagi_moe_combine_bwd(
        mu_g.data_ptr(), jcb_g.data_ptr(), mu_y.data_ptr(), expert.data_ptr(), slot.data_ptr(),
        delta_mu.data_ptr(), delta_var.data_ptr(), T, k, R, N, num_experts, dmu_y.data_ptr(),
        dvar_y.data_ptr(), dmu_s.data_ptr(), dvar_s.data_ptr(), _raw_stream(dev)))
    return dmu_y, dvar_y, dmu_s, dvar_s


def moe_gather_bwd(delta_mu_r, delta_var_r, slot, jcb=None, res_mu=None, res_var=None):
    """Row innovations [R, K] back to the tokens: jcb * (sum over the token's rows + res), and
    jcb^2 for the variances, [T, K]."""
    _pair(res_mu, res_var, ("res_mu", "res_var"))
    T, k = _dims("slot", slot, 2)
    R, K = _dims("delta_mu_r", delta_mu_r, 2)
    dev = _device(delta_mu_r)
    if not (_fits(dev, _I, (T, k), slot) and _fits(dev, _F, (R, K), delta_mu_r, delta_var_r) and
            _fits(dev, _F, (T, K), jcb, res_mu, res_var)):
        _explain(slot=(slot, (T, k), _I), delta_mu_r=(delta_mu_r, (R, K), _F),
                 delta_var_r=(delta_var_r, (R, K), _F), jcb=(jcb, (T, K), _F),
                 res_mu=(res_mu, (T, K), _F), res_var=(res_var, (T, K), _F))
    dmu, dvar = _new(delta_mu_r, 2, T, K)
    capi.check(capi.lib.tagi_moe_gather_bwd(
        delta_mu_r.data_ptr(), delta_var_r.data_ptr(), slot.data_ptr(), _at(jcb), _at(res_mu),
        _at(res_var), T, k, R, K, dmu.data_ptr(), dvar.data_ptr(), _raw_stream(dev)))
    return dmu, dvar
