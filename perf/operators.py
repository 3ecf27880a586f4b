"""The operators of a pre-norm mixture-of-experts feed-forward block in TAGI form, as
workloads: every unit, weight and gate is a Gaussian, so each operator carries means and
variances forward and innovations (delta_mu, delta_var) backward, all in fp32.

  norm      layer norm over the features of each row ("fwd"), with its backward pass and the
            reductions of the weight and bias innovations ("train")
  experts   Linear layers grouped by expert, rows sorted by expert with ragged group sizes:
            forward ("fwd"), all of the backward pass ("bwd"), or both ("train")
  route     choice of the top_k experts per token, their gates, and the plan of the rows
  combine   the gated sum of the experts' outputs ("fwd"), with its backward pass ("train")

Sizes are those of the repository's Linear workloads (4096 features, batches from a few
samples to thousands) and generic odd ones.
"""
import math

import torch

own = False

EPS = 1e-5


def listed():
    return [
        # one token of a served model through a norm layer
        dict(name="norm_token", op="norm", phase="fwd", rows=1, n=4096),
        # a training batch of odd size
        dict(name="norm_train_odd", op="norm", phase="train", rows=999, n=1023),
        # a training batch of long sequences
        dict(name="norm_train_large", op="norm", phase="train", rows=16384, n=4096),
        # one served token that visits two of eight experts
        dict(name="experts_token", op="experts", phase="fwd", tokens=1, top_k=2, experts=8,
             K=4096, N=4096, gather=True),
        # one decoding step of 32 users
        dict(name="experts_decode", op="experts", phase="fwd", tokens=32, top_k=2, experts=16,
             K=2048, N=4096, gather=True),
        # a prompt: thousands of rows, gathered from their tokens
        dict(name="experts_prompt", op="experts", phase="fwd", tokens=4096, top_k=2, experts=8,
             K=2048, N=4096, gather=True),
        # the backward pass of an expert's second layer in training
        dict(name="experts_bwd_large", op="experts", phase="bwd", tokens=4096, top_k=2, experts=8,
             K=4096, N=2048, gather=False),
        # a small training batch, odd sizes everywhere
        dict(name="experts_train_odd", op="experts", phase="train", tokens=259, top_k=3, experts=6,
             K=301, N=415, gather=True),
        # the router of a decoding step, some of the batch's places empty
        dict(name="route_step", op="route", tokens=32, experts=16, top_k=2, padded=5),
        # the router of a training batch with many experts
        dict(name="route_large", op="route", tokens=16384, experts=64, top_k=4, padded=0),
        # the gated sum of a decoding step
        dict(name="combine_step", op="combine", phase="fwd", tokens=32, top_k=2, experts=16,
             N=4096, padded=5),
        # the gated sum of a training batch and its backward pass
        dict(name="combine_train", op="combine", phase="train", tokens=8192, top_k=2, experts=8,
             N=4096, padded=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "experts", "experts", "route", "combine"])
    if op == "norm":
        n = _log(rng, 2, 8192)
        return dict(op=op, phase=rng.choice(["fwd", "train"]),
                    rows=_log(rng, 1, min(65536, 16384 * 4096 // n)), n=n)
    if op == "experts":
        experts = _log(rng, 1, 32)
        top_k = rng.randint(1, min(4, experts))
        K, N = _log(rng, 16, 4096), _log(rng, 16, 4096)
        while experts * K * N > 8 * 4096 * 4096:
            K, N = max(16, K // 2), max(16, N // 2)
        most = min(8192, 8192 * 2048 * 4096 // (K * N))
        phase = rng.choice(["fwd", "bwd", "train"])
        tokens = max(1, _log(rng, 1, most) // top_k // (2 if phase == "train" else 1))
        return dict(op=op, phase=phase, tokens=tokens, top_k=top_k, experts=experts, K=K, N=N,
                    gather=rng.random() < 0.5)
    if op == "route":
        experts = _log(rng, 1, 256)
        tokens = _log(rng, 1, min(65536, 16384 * 64 // experts))
        return dict(op=op, tokens=tokens, experts=experts, top_k=rng.randint(1, min(8, experts)),
                    padded=rng.randint(0, tokens // 4))
    experts = _log(rng, 2, 64)
    top_k = rng.randint(1, min(4, experts))
    N = _log(rng, 1, 8192)
    tokens = _log(rng, 1, min(32768, 8192 * 2 * 4096 // (N * top_k)))
    return dict(op=op, phase=rng.choice(["fwd", "train"]), tokens=tokens, top_k=top_k,
                experts=experts, N=N, padded=rng.randint(0, tokens // 4))


# ---- inputs ---------------------------------------------------------------------------------

class _Maker:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, scale=1.0):
        return torch.randn(shape, generator=self.g, device="cuda").mul_(scale)

    def uniform(self, lo, hi, *shape):
        return torch.rand(shape, generator=self.g, device="cuda").mul_(hi - lo).add_(lo)


def _scores(m, tokens, experts, padded):
    """Mean scores with popular and unpopular experts; the last `padded` tokens are empty
    places of the batch, which may go to no expert."""
    s = m.normal(tokens, experts) + m.normal(experts, scale=0.3)
    if padded:
        s[tokens - padded:] = -math.inf
    return s


def _chosen(scores, top_k):
    """[T][k] experts by falling score (ties: lowest index), -1 where none may be chosen."""
    v, i = torch.sort(scores, dim=1, descending=True, stable=True)
    return torch.where(v[:, :top_k] > -math.inf, i[:, :top_k], -1)


def _plan(expert, experts):
    """offsets [E+1], the token of every row and the row of every choice, rows sorted by
    expert and then by token; -1 in places that hold no row."""
    T, k = expert.shape
    e = torch.where(expert < 0, experts, expert).reshape(-1)
    order = torch.argsort(e, stable=True)
    slot = torch.empty_like(order)
    slot[order] = torch.arange(T * k, device=e.device)
    count = (e[:, None] == torch.arange(experts, device=e.device)).sum(0)
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=e.device)
    offsets[1:] = torch.cumsum(count, 0)
    row = torch.arange(T * k, device=e.device)
    token = torch.where(row < offsets[-1], order // k, -1)
    slot = torch.where(e < experts, slot, -1).reshape(T, k)
    return offsets.int(), token.int(), slot.int()


def prepare(case, seed):
    m = _Maker(seed)
    op, s = case["op"], dict(case)
    if op == "norm":
        rows, n = case["rows"], case["n"]
        s.update(mu_w=1 + m.normal(n, scale=0.1), var_w=m.uniform(0.01, 0.1, n),
                 mu_b=m.normal(n, scale=0.1), var_b=m.uniform(0.01, 0.1, n),
                 mu_a=m.normal(rows, n) + m.normal(rows, 1), var_a=m.uniform(0.01, 0.5, rows, n))
        if case["phase"] == "train":
            s.update(jcb=m.uniform(0.0, 1.0, rows, n), dmu=m.normal(rows, n, scale=0.1),
                     dvar=-m.uniform(0.0, 1e-2, rows, n))
    elif op == "experts":
        T, k, E, K, N = (case[x] for x in ("tokens", "top_k", "experts", "K", "N"))
        R = T * k
        offsets, token, _ = _plan(_chosen(_scores(m, T, E, 0), k), E)
        s.update(offsets=offsets, rows=token if case["gather"] else None,
                 cap=int((offsets[1:] - offsets[:-1]).max()))
        held = T if case["gather"] else R
        s.update(mu_w=m.normal(E, N, K, scale=K ** -0.5), var_w=m.uniform(0.5 / K, 1.5 / K, E, N, K),
                 mu_b=m.normal(E, N, scale=0.5), var_b=m.uniform(0.5 / K, 1.5 / K, E, N),
                 mu_a=m.normal(held, K), var_a=m.uniform(0.01, 0.1, held, K))
        if case["phase"] != "fwd":
            s.update(jcb=m.uniform(0.0, 1.0, R, K), dmu=m.normal(R, N, scale=0.1),
                     dvar=-m.uniform(0.0, 1e-3, R, N))
    elif op == "route":
        T, E = case["tokens"], case["experts"]
        s.update(mu_s=_scores(m, T, E, case["padded"]), var_s=m.uniform(0.01, 0.5, T, E))
    else:
        T, k, E, N = (case[x] for x in ("tokens", "top_k", "experts", "N"))
        mu_s = _scores(m, T, E, case["padded"])
        expert = _chosen(mu_s, k)
        offsets, token, slot = _plan(expert, E)
        g = torch.softmax(torch.where(expert < 0, 0.0, torch.gather(mu_s, 1, expert.clamp(min=0))), 1)
        g = torch.where(expert < 0, 0.0, g)
        jcb_g = g * (1 - g)
        s.update(expert=expert.int(), slot=slot, mu_g=g.contiguous(), jcb_g=jcb_g.contiguous(),
                 var_g=(jcb_g * jcb_g * m.uniform(0.01, 0.5, T, k)).contiguous(),
                 mu_y=m.normal(T * k, N), var_y=m.uniform(0.01, 0.5, T * k, N))
        if case["phase"] == "train":
            s.update(dmu=m.normal(T, N, scale=0.1), dvar=-m.uniform(0.0, 1e-2, T, N))
    return s


# ---- the framework's calls ------------------------------------------------------------------

def _run_own(s):
    import cutagi_amd.functional as F
    op, out = s["op"], {}
    if op == "norm":
        mu_z, var_z, mu_s, var_s = F.layernorm_fwd(s["mu_w"], s["var_w"], s["mu_b"], s["var_b"],
                                                   s["mu_a"], s["var_a"], EPS)
        out.update(mu_z=mu_z, var_z=var_z, mu_s=mu_s, var_s=var_s)
        if s["phase"] == "train":
            names = ("dz_mu", "dz_var", "dw_mu", "dw_var", "db_mu", "db_var")
            out.update(zip(names, F.layernorm_bwd(s["mu_w"], s["var_w"], s["var_b"], s["mu_a"],
                                                  s["jcb"], mu_s, var_s, s["dmu"], s["dvar"], EPS)))
    elif op == "experts":
        if s["phase"] != "bwd":
            out["mu_z"], out["var_z"] = F.grouped_linear_fwd(
                s["mu_w"], s["var_w"], s["mu_b"], s["var_b"], s["mu_a"], s["var_a"], s["offsets"],
                rows=s["rows"])
        if s["phase"] != "fwd":
            names = ("dz_mu", "dz_var", "dw_mu", "dw_var", "db_mu", "db_var")
            out.update(zip(names, F.grouped_linear_bwd(
                s["mu_w"], s["var_w"], s["var_b"], s["mu_a"], s["jcb"], s["dmu"], s["dvar"],
                s["offsets"], rows=s["rows"])))
    elif op == "route":
        r = F.moe_route(s["mu_s"], s["var_s"], s["top_k"])
        out.update(expert=r.expert, mu_g=r.mu_g, var_g=r.var_g, jcb_g=r.jcb_g, offsets=r.offsets,
                   token=r.token, slot=r.slot)
    else:
        out["mu_z"], out["var_z"] = F.moe_combine_fwd(s["mu_g"], s["var_g"], s["mu_y"], s["var_y"],
                                                      s["slot"])
        if s["phase"] == "train":
            # innovations of rows that no token holds are left as they were: zeros here
            rows = (torch.zeros if s["padded"] else torch.empty)(
                (2,) + s["mu_y"].shape, device=s["mu_y"].device)
            out.update(zip(("dy_mu", "dy_var", "ds_mu", "ds_var"), F.moe_combine_bwd(
                s["mu_g"], s["jcb_g"], s["mu_y"], s["expert"], s["slot"], s["dmu"], s["dvar"],
                s["experts"], out=(rows[0], rows[1]))))
    return out


# ---- the plain forms ------------------------------------------------------------------------

def _plain_norm(s):
    n = s["n"]
    mean = s["mu_a"].mean(1)
    d = s["mu_a"] - mean[:, None]
    var = ((d * d).sum(1) + s["var_a"].sum(1)) / (n - 1)
    inv = (1.0 / torch.sqrt(var + EPS))[:, None]
    mw, vw = s["mu_w"], s["var_w"]
    x = inv * d
    out = dict(mu_z=x * mw + s["mu_b"],
               var_z=inv * inv * s["var_a"] * (mw * mw + vw) + vw * x * x + s["var_b"],
               mu_s=mean, var_s=var)
    if s["phase"] == "train":
        t = inv * mw * s["jcb"]
        out.update(dz_mu=t * s["dmu"], dz_var=t * t * s["dvar"], dw_mu=vw * (x * s["dmu"]).sum(0),
                   dw_var=vw * vw * (x * x * s["dvar"]).sum(0), db_mu=s["var_b"] * s["dmu"].sum(0),
                   db_var=s["var_b"] * s["var_b"] * s["dvar"].sum(0))
    return out


def _plain_experts(s):
    off, cap, R = s["offsets"].long(), s["cap"], s["tokens"] * s["top_k"]
    dev = off.device
    # every group padded to the largest one, so that the experts are one batched product
    place = off[:-1, None] + torch.arange(cap, device=dev)
    held = (place < off[1:, None])[..., None]
    place = place.clamp(max=R - 1)
    row = torch.arange(R, device=dev)
    group = torch.searchsorted(off[1:].contiguous(), row, right=True)
    back = group * cap + row - off[group]
    source = place if s["rows"] is None else s["rows"].long()[place]
    mw, vw = s["mu_w"], s["var_w"]
    x = torch.where(held, s["mu_a"][source], 0.0)
    out = {}
    if s["phase"] != "bwd":
        v = torch.where(held, s["var_a"][source], 0.0)
        mu = torch.bmm(x, mw.transpose(1, 2)) + s["mu_b"][:, None]
        var = torch.bmm(v + x * x, vw.transpose(1, 2)) + torch.bmm(v, (mw * mw).transpose(1, 2))
        var = var + s["var_b"][:, None]
        out.update(mu_z=mu.flatten(0, 1)[back], var_z=var.flatten(0, 1)[back])
    if s["phase"] != "fwd":
        dm = torch.where(held, s["dmu"][place], 0.0)
        dv = torch.where(held, s["dvar"][place], 0.0)
        j = s["jcb"]
        out.update(dz_mu=torch.bmm(dm, mw).flatten(0, 1)[back] * j,
                   dz_var=torch.bmm(dv, mw * mw).flatten(0, 1)[back] * j * j,
                   dw_mu=torch.bmm(dm.transpose(1, 2), x) * vw,
                   dw_var=torch.bmm(dv.transpose(1, 2), x * x) * vw * vw,
                   db_mu=dm.sum(1) * s["var_b"], db_var=dv.sum(1) * s["var_b"] * s["var_b"])
    return out


def _plain_route(s):
    expert = _chosen(s["mu_s"], s["top_k"])
    offsets, token, slot = _plan(expert, s["experts"])
    ok = expert >= 0
    at = expert.clamp(min=0)
    mu = torch.where(ok, torch.gather(s["mu_s"], 1, at), -math.inf)
    # the first choice has the largest score; a token without one gets gates of zero
    e = torch.where(ok, torch.exp(mu - mu[:, :1]), 0.0)
    g = torch.where(ok, e / e.sum(1, keepdim=True), 0.0)
    jcb = g * (1 - g)
    return dict(expert=expert.int(), mu_g=g,
                var_g=torch.where(ok, jcb * jcb * torch.gather(s["var_s"], 1, at), 0.0), jcb_g=jcb,
                offsets=offsets, token=token, slot=slot)


def _plain_combine(s):
    slot = s["slot"].long()
    ok = (slot >= 0)[..., None]
    at = slot.clamp(min=0)
    g, vg = s["mu_g"][..., None], s["var_g"][..., None]
    y = torch.where(ok, s["mu_y"][at], 0.0)
    v = torch.where(ok, s["var_y"][at], 0.0)
    out = dict(mu_z=(g * y).sum(1), var_z=((g * g + vg) * v + vg * y * y).sum(1))
    if s["phase"] == "train":
        T, k = slot.shape
        R = T * k
        dmu, dvar, j = s["dmu"][:, None], s["dvar"][:, None], s["jcb_g"]
        # row -> choice; places that hold no row point at an extra choice of zeros
        choice = torch.full((R + 1,), R, dtype=torch.int64, device=slot.device)
        choice[torch.where(slot < 0, R, slot).reshape(-1)] = torch.arange(R, device=slot.device)
        choice = choice[:R]
        real, choice = (choice < R)[:, None], choice.clamp(max=R - 1)
        gate = s["mu_g"].reshape(-1)[choice][:, None]
        out.update(dy_mu=torch.where(real, gate * s["dmu"][choice // k], 0.0),
                   dy_var=torch.where(real, gate * gate * s["dvar"][choice // k], 0.0))
        to = torch.where(s["expert"] < 0, s["experts"], s["expert"]).long()
        ds = torch.zeros((2, T, s["experts"] + 1), device=slot.device)
        ds[0].scatter_(1, to, j * (y * dmu).sum(2))
        ds[1].scatter_(1, to, j * j * (y * y * dvar).sum(2))
        out.update(ds_mu=ds[0, :, :-1].contiguous(), ds_var=ds[1, :, :-1].contiguous())
    return out


def run(state):
    if own:
        return _run_own(state)
    return dict(norm=_plain_norm, experts=_plain_experts, route=_plain_route,
                combine=_plain_combine)[state["op"]](state)


# ---- what the operators cannot do without ---------------------------------------------------

def work(case):
    op = case["op"]
    if op == "norm":
        size, n = case["rows"] * case["n"], case["n"]
        train = case["phase"] == "train"
        # (mu_a, var_a) -> (mu_z, var_z); (jcb, dmu, dvar) -> (dmu, dvar) and the parameters
        return dict(bytes=4 * (size * (9 if train else 4) + n * (8 if train else 4) + 2 * case["rows"]),
                    flops=size * (32 if train else 18))
    if op == "experts":
        T, k, E, K, N = (case[x] for x in ("tokens", "top_k", "experts", "K", "N"))
        R, held = T * k, T if case["gather"] else T * k
        used = min(E, R)          # experts that can have rows
        if case["phase"] == "fwd":
            return dict(bytes=8 * (used * N * (K + 1) + held * K + R * N), flops=6 * R * K * N)
        if case["phase"] == "bwd":   # mu_w of the used, var_w of all experts, mu_a, jcb, deltas
            return dict(bytes=4 * (used * N * K + E * N * (3 * K + 3) + held * K + 3 * R * K + 2 * R * N),
                        flops=8 * R * K * N)
        return dict(bytes=4 * (used * N * K + E * N * (3 * K + 4) + 2 * held * K + 3 * R * K + 4 * R * N),
                    flops=14 * R * K * N)
    T, k, E = case["tokens"], case["top_k"], case["experts"]
    if op == "route":
        return dict(bytes=4 * (T * E + T * k * 7 + E + 1), flops=T * E * k)
    N = case["N"]
    if case["phase"] == "fwd":
        return dict(bytes=4 * (2 * T * k * (N + 1) + T * k + 2 * T * N), flops=8 * T * k * N)
    return dict(bytes=4 * (2 * T * k * N + 5 * T * k + 4 * T * N + 2 * T * k * N + 2 * T * E),
                flops=16 * T * k * N)


# ---- 64 bits --------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    f = {k: (v.double() if torch.is_tensor(v) and v.is_floating_point() else v) for k, v in s.items()}
    return dict(norm=_exact_norm, experts=_exact_experts, route=_exact_route,
                combine=_exact_combine)[case["op"]](f)


def _exact_norm(f):
    n, a = f["n"], f["mu_a"]
    mean = a.sum(1) / n
    centred = a - mean.unsqueeze(1)
    var = (centred.square().sum(1) + f["var_a"].sum(1)) / (n - 1)
    scale2 = 1 / (var + EPS).unsqueeze(1)
    scale = scale2.sqrt()
    out = dict(mu_z=centred * scale * f["mu_w"] + f["mu_b"],
               var_z=scale2 * (f["var_a"] * (f["mu_w"].square() + f["var_w"]) +
                               f["var_w"] * centred.square()) + f["var_b"], mu_s=mean, var_s=var)
    if f["phase"] == "train":
        slope = f["mu_w"] * scale * f["jcb"]
        unit = centred * scale
        out.update(dz_mu=f["dmu"] * slope, dz_var=f["dvar"] * slope.square(),
                   dw_mu=f["var_w"] * torch.einsum("bi,bi->i", unit, f["dmu"]),
                   dw_var=f["var_w"].square() * torch.einsum("bi,bi->i", unit.square(), f["dvar"]),
                   db_mu=f["var_b"] * f["dmu"].sum(0), db_var=f["var_b"].square() * f["dvar"].sum(0))
    return out


def _exact_experts(f):
    ends = f["offsets"].tolist()
    a, v = f["mu_a"], f["var_a"]
    if f["rows"] is not None:
        a, v = a[f["rows"].long()], v[f["rows"].long()]
    parts = {}

    def keep(**tensors):
        for name, t in tensors.items():
            parts.setdefault(name, []).append(t)

    for e in range(f["experts"]):
        r = slice(ends[e], ends[e + 1])
        w, q = f["mu_w"][e], f["var_w"][e]
        if f["phase"] != "bwd":
            keep(mu_z=a[r] @ w.T + f["mu_b"][e],
                 var_z=a[r].square() @ q.T + v[r] @ (w.square() + q).T + f["var_b"][e])
        if f["phase"] != "fwd":
            dm, dv, j = f["dmu"][r], f["dvar"][r], f["jcb"][r]
            keep(dz_mu=j * (dm @ w), dz_var=j.square() * (dv @ w.square()),
                 dw_mu=q * (dm.T @ a[r]), dw_var=q.square() * (dv.T @ a[r].square()),
                 db_mu=f["var_b"][e] * dm.sum(0), db_var=f["var_b"][e].square() * dv.sum(0))
    return {name: (torch.cat if name[:2] in ("mu", "va", "dz") else torch.stack)(p)
            for name, p in parts.items()}


def _exact_route(f):
    scores = f["mu_s"].cpu()
    T, E, k = f["tokens"], f["experts"], f["top_k"]
    order = torch.argsort(-scores, dim=1, stable=True)[:, :k]
    top = torch.gather(scores, 1, order)
    ok = torch.isfinite(top)
    expert = torch.where(ok, order, torch.full_like(order, -1))
    weight = torch.where(ok, (top - top[:, :1].nan_to_num(neginf=0.0)).exp(), torch.zeros_like(top))
    total = weight.sum(1, keepdim=True)
    gate = weight / torch.where(total > 0, total, torch.ones_like(total))
    slope = weight * (total - weight) / torch.where(total > 0, total, torch.ones_like(total)).square()
    member = torch.zeros((E, T), dtype=torch.int64)
    t, j = torch.nonzero(ok, as_tuple=True)
    member[expert[t, j], t] = 1
    offsets = torch.zeros(E + 1, dtype=torch.int64)
    offsets[1:] = torch.cumsum(member.sum(1), 0)
    rank = (torch.cumsum(member.reshape(-1), 0) - 1).reshape(E, T)
    slot = torch.full((T, k), -1, dtype=torch.int64)
    slot[t, j] = rank[expert[t, j], t]
    token = torch.full((T * k,), -1, dtype=torch.int64)
    token[slot[t, j]] = t
    return dict(expert=expert.int(), mu_g=gate,
                var_g=slope.square() * torch.gather(f["var_s"].cpu(), 1, order) * ok, jcb_g=slope,
                offsets=offsets.int(), token=token.int(), slot=slot.int())


def _exact_combine(f):
    slot, k = f["slot"].long(), f["top_k"]
    T, N = f["tokens"], f["N"]
    zero = torch.zeros((T, N), dtype=torch.float64, device=slot.device)
    out = dict(mu_z=zero.clone(), var_z=zero.clone())
    if f["phase"] == "train":
        out.update(dy_mu=torch.zeros_like(f["mu_y"]), dy_var=torch.zeros_like(f["mu_y"]),
                   ds_mu=torch.zeros((T, f["experts"]), dtype=torch.float64, device=slot.device))
        out["ds_var"] = out["ds_mu"].clone()
    for j in range(k):
        t = torch.nonzero(slot[:, j] >= 0)[:, 0]
        r, g, vg = slot[t, j], f["mu_g"][t, j].unsqueeze(1), f["var_g"][t, j].unsqueeze(1)
        y, v = f["mu_y"][r], f["var_y"][r]
        out["mu_z"][t] += g * y
        out["var_z"][t] += g.square() * v + vg * (v + y.square())
        if f["phase"] == "train":
            out["dy_mu"][r], out["dy_var"][r] = g * f["dmu"][t], g.square() * f["dvar"][t]
            e, slope = f["expert"][t, j].long(), f["jcb_g"][t, j]
            out["ds_mu"][t, e] = slope * torch.einsum("tn,tn->t", y, f["dmu"][t])
            out["ds_var"][t, e] = slope.square() * torch.einsum("tn,tn->t", y.square(), f["dvar"][t])
    return out
