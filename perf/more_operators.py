"""Routing to experts, the rows between tokens and experts, and low-rank adapters, as cases that a timing harness can run.

`kind` of a case says which operators it goes through:

    route     route_experts: the router's logits become weights, experts and the pairs' order by expert
              (train: grad.route_experts and its backward pass)
    rows      dispatch_rows and combine_rows: activations to the experts' order, the experts' results back to the tokens
              (train: the forms in grad, and both backward passes)
    adapters  group_rows once, then add_adapters beside both projections of an MLP (K to N, N to K)
              (train: grad.add_adapters beside the first one and its backward pass)

`own` says who computes: the framework's operators, or (False) their plain forms below, which follow the formulas in
32 bits (the routing's order of keys in 64) and round once at the end.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_INF = float("inf")


def _route(T, E, top, scoring, dtype, renormalize=True, bias=False, groups=1, top_groups=1, group_best=1, scale=1.0, train=False):
    return {"kind": "route", "T": T, "E": E, "top": top, "scoring": scoring, "dtype": dtype, "renormalize": renormalize, "bias": bias,
            "groups": groups, "top_groups": top_groups, "group_best": group_best, "scale": scale, "train": train}


def _rows(T, E, top, D, dtype, train=False):
    return {"kind": "rows", "T": T, "E": E, "top": top, "D": D, "dtype": dtype, "train": train}


def _adapters(T, requests, L, rank, N, K, dtype, train=False):
    return {"kind": "adapters", "T": T, "requests": requests, "L": L, "rank": rank, "N": N, "K": K, "dtype": dtype, "train": train}


def listed():
    return [
        # four sequences decoded together, top-2 of 8 experts: the smallest call of a decode loop
        {"name": "route 4 tokens", **_route(4, 8, 2, "softmax", "f32")},
        # many narrow experts in groups, kept in balance by a bias: a server's decode batch
        {"name": "route 64 tokens groups", **_route(64, 256, 8, "sigmoid", "f32", bias=True, groups=8, top_groups=4, group_best=2, scale=2.5)},
        # the same router over long prompts
        {"name": "route 8192 tokens groups", **_route(8192, 256, 8, "sigmoid", "f32", bias=True, groups=8, top_groups=4, group_best=2, scale=2.5)},
        # a router being trained: probabilities over all experts, whose gradient is dense
        {"name": "route train 16384 tokens", **_route(16384, 128, 8, "softmax", "bf16", renormalize=False, train=True)},
        # half precision, an odd number of tokens, a number of experts that is no power of two
        {"name": "route train 1531 tokens f16", **_route(1531, 60, 4, "softmax", "f16", train=True)},
        # four sequences decoded together through an expert layer of this repository's benchmark
        {"name": "rows 4 tokens", **_rows(4, 8, 2, 4096, "bf16")},
        # that layer being trained
        {"name": "rows train 4096 tokens", **_rows(4096, 8, 2, 4096, "bf16", train=True)},
        # many experts per token, rows that are not whole vectors, half precision
        {"name": "rows train 1531 tokens f16", **_rows(1531, 64, 6, 2047, "f16", train=True)},
        # one request with its adapter
        {"name": "adapters 1 row", **_adapters(1, 1, 8, 16, 14336, 4096, "bf16")},
        # a decode batch whose requests mostly have adapters of their own, half precision, a rank that is no power of two
        {"name": "adapters 57 rows f16", **_adapters(57, 57, 40, 20, 11008, 4096, "f16")},
        # five prompts with different adapters
        {"name": "adapters 4096 rows", **_adapters(4096, 5, 16, 64, 14336, 4096, "bf16")},
        # adapters being trained, four of them in one batch
        {"name": "adapters train 2048 rows", **_adapters(2048, 8, 4, 16, 14336, 4096, "bf16", train=True)},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges: one token to many, 4 to 512 experts, ranks from 4 to 128, widths that are mostly whole
    64s and sometimes any number, every type and both directions."""
    most = {key: max(work(c)[key] for c in listed()) for key in ("bytes", "flops")}
    while True:
        kind = rng.choice(["route", "rows", "adapters"])
        train = rng.random() < 0.4
        if kind == "route":
            groups = rng.choice([1, 1, 2, 4, 8])
            E = groups * _log_int(rng, 4, 512 // groups)
            top_groups = rng.randint(1, groups)
            top = rng.randint(1, min(16, E // groups * top_groups))
            c = _route(_log_int(rng, 1, 16384), E, top, rng.choice(["softmax", "sigmoid"]), rng.choice(["f32", "bf16", "f16"]),
                       rng.random() < 0.6, rng.random() < 0.5, groups, top_groups, rng.choice([1, 2]), rng.choice([1.0, 2.5]), train)
        elif kind == "rows":
            E = _log_int(rng, 2, 128)
            D = _log_int(rng, 128, 8192)
            c = _rows(_log_int(rng, 1, 8192), E, rng.randint(1, min(E, 8)), D if rng.random() < 0.25 else D // 64 * 64,
                      rng.choice(["bf16", "bf16", "f16", "f32"]), train)
        else:
            N, K = _log_int(rng, 256, 14336), _log_int(rng, 256, 14336)
            if rng.random() < 0.75:
                N, K = N // 64 * 64, K // 64 * 64
            T = _log_int(rng, 1, 8192)
            rank = rng.choice([4, 8, 16, 16, 32, 64, 128]) if rng.random() < 0.8 else rng.randint(4, 128)
            c = _adapters(T, min(T, _log_int(rng, 1, 128)), _log_int(rng, 1, 64), rank, N, K, rng.choice(["bf16", "bf16", "f16"]), train)
        if all(work(c)[key] <= most[key] for key in most):
            return c


def _bytes(dtype):
    return 4 if dtype == "f32" else 2


def work(case):
    """Bytes that have to be read and written once, and operations."""
    b, T = _bytes(case["dtype"]), case["T"]
    if case["kind"] == "route":
        E, pairs = case["E"], T * case["top"]
        n = T * E * b + 16 * pairs + 4 * E + (4 * E if case["bias"] else 0)
        flops = 4 * T * E
        if case["train"]:   # the weights' gradient comes in, the logits' goes out, which reads all of them where the softmax is over all
            n += 4 * pairs + T * E * b + (T * E * b if case["scoring"] == "softmax" and not case["renormalize"] else 0)
            flops *= 2
        return {"bytes": n, "flops": flops}
    if case["kind"] == "rows":
        tokens, rows = T * case["D"] * b, T * case["top"] * case["D"] * b
        ids = 8 * T * case["top"]
        n, flops = 2 * (tokens + rows) + 2 * ids, 2 * T * case["top"] * case["D"]
        if case["train"]:   # d x from d xs; d ys and d weights from dy and ys
            n += (tokens + rows) + (tokens + 2 * rows) + 3 * ids
            flops *= 4
        return {"bytes": n, "flops": flops}
    N, K, r = case["N"], case["K"], case["rank"]
    used = min(case["L"], case["requests"])
    if case["train"]:
        # forward reads x, y, the adapters and writes the sum; backward reads dy, x, the adapters and writes dx and their gradients
        n = T * (K + 2 * N) * b + T * (2 * K + N) * b + 2 * used * r * (K + N) * b + case["L"] * r * (K + N) * b
        return {"bytes": n, "flops": 6 * T * r * (K + N)}
    n = T * (K + 2 * N) * b + T * (N + 2 * K) * b + 2 * used * r * (K + N) * b
    return {"bytes": n, "flops": 4 * T * r * (K + N)}


# ------------------------------------------------------------------------------------------------ inputs
def _pairs_by_expert(experts, E):
    """Pairs (token, choice) in the experts' order: sizes, every pair's place, the pair at every place."""
    flat = experts.flatten().long()
    order = flat.argsort(stable=True)
    places = torch.empty_like(order)
    places[order] = torch.arange(len(order), device=order.device)
    sizes = torch.bincount(flat, minlength=E)
    return sizes.int(), places.int().reshape(experts.shape), order.int()


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dt, T = _DTYPES[case["dtype"]], case["T"]

    def normal(shape, std, dtype=dt):
        return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)

    st = {"case": case}
    if case["kind"] == "route":
        E = case["E"]
        # some experts are asked for more often than others; the bias, learned from their load, pulls the other way
        liking = torch.randn(E, generator=gen, device="cuda")
        st["logits"] = (torch.randn((T, E), generator=gen, device="cuda") * 1.5 + 0.5 * liking).to(dt)
        st["bias"] = -0.05 * liking + 0.02 * torch.randn(E, generator=gen, device="cuda") if case["bias"] else None
        if case["train"]:
            st["dw"] = normal((T, case["top"]), 1.0, torch.float32)
            st["logits"].requires_grad_()
        return st
    if case["kind"] == "rows":
        E, top, D = case["E"], case["top"], case["D"]
        p = torch.rand(E, generator=gen, device="cuda") + 0.25
        experts = torch.multinomial(p.expand(T, E), top, generator=gen)
        w = torch.rand((T, top), generator=gen, device="cuda") + 0.1
        st["weights"], st["experts"] = w / w.sum(-1, keepdim=True), experts.int()
        st["sizes"], st["places"], st["order"] = _pairs_by_expert(experts, E)
        st["x"], st["y"] = normal((T, D), 1.0), normal((T * top, D), 1.0)
        if case["train"]:
            st["dxs"], st["dy"] = normal((T * top, D), 0.1), normal((T, D), 0.1)
            for name in ("x", "y", "weights"):
                st[name].requires_grad_()
        return st
    N, K, r, L, n = case["N"], case["K"], case["rank"], case["L"], case["requests"]
    # every request has its adapter, one in eight has none; its rows lie together
    g = torch.Generator().manual_seed(seed)
    adapter = torch.randint(0, L, (n,), generator=g)
    if n > 1:
        adapter[torch.rand(n, generator=g) < 0.125] = -1
    cuts = torch.cat((torch.tensor([0]), torch.randperm(T - 1, generator=g)[:n - 1].sort().values + 1, torch.tensor([T])))
    st["ids"] = adapter.repeat_interleave(cuts.diff()).cuda()
    st["scales"] = (torch.rand(L, generator=gen, device="cuda") + 0.5)
    st["a"], st["b"] = normal((L, r, K), K ** -0.5), normal((L, N, r), r ** -0.5)
    st["x"], st["y"] = normal((T, K), 1.0), normal((T, N), 1.0)
    if case["train"]:
        st["dy"] = normal((T, N), 0.1)
        for name in ("x", "y", "a", "b"):
            st[name].requires_grad_()
    else:
        st["a2"], st["b2"] = normal((L, r, N), N ** -0.5), normal((L, K, r), r ** -0.5)
        st["x2"], st["y2"] = normal((T, N), 1.0), normal((T, K), 1.0)
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _choose(case, logits, bias):
    """Experts [T, top] by falling key, -1 for those that are off: the logits' order, with a bias that of score + bias, in 64 bits,
    since two keys next to each other decide which expert a token gets."""
    E, G = case["E"], case["groups"]
    l = logits.double()
    score = torch.softmax(l, -1) if case["scoring"] == "softmax" else torch.sigmoid(l)
    key = l if bias is None else torch.where(l == -_INF, -_INF, score + bias.double())
    if G > 1:
        best, at = key.unflatten(-1, (G, E // G)).topk(case["group_best"], -1)
        rank = best[..., 0]
        if case["group_best"] == 2:
            added = best if bias is not None else score.unflatten(-1, (G, E // G)).gather(-1, at)
            rank = torch.where(rank == -_INF, -_INF, torch.where(best == -_INF, 0.0, added).sum(-1))
        kept = rank.sort(dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        on = torch.zeros_like(rank, dtype=torch.bool).scatter_(1, kept, True)
        key = torch.where(on.repeat_interleave(E // G, 1), key, -_INF)
    value, expert = (v[:, :case["top"]] for v in key.sort(dim=-1, descending=True, stable=True))
    return torch.where(value == -_INF, -1, expert)


def _plain_route(st):
    case = st["case"]
    l = st["logits"].detach().float()
    experts = _choose(case, st["logits"].detach(), st["bias"])
    has = experts >= 0
    e = experts.clamp_min(0)
    if case["scoring"] == "softmax":
        z = torch.exp(l - l.amax(-1, keepdim=True))
        score = z / z.sum(-1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-l))
    w = torch.where(has, score.gather(1, e), 0.0)
    total = w.sum(-1, keepdim=True)
    q = w / total if case["renormalize"] else w
    out = {"weights": q * case["scale"], "experts": experts.int()}
    last = torch.where(has, experts, case["E"])   # pairs without an expert come last
    sizes, places, order = _pairs_by_expert(last, case["E"] + 1)
    rows = torch.arange(len(order), device=order.device) < sizes[:-1].sum()
    out["sizes"], out["places"] = sizes[:-1], torch.where(has, places, -1).int()
    out["order"] = torch.where(rows, order, -1 - order).int()
    if case["train"]:
        g = st["dw"] * case["scale"]
        if case["renormalize"]:
            g = (g - (g * q).sum(-1, keepdim=True)) / total   # with respect to the chosen scores
        if case["scoring"] == "softmax":
            dense = torch.zeros_like(l).scatter_add_(1, e, torch.where(has, g, 0.0))
            dl = score * (dense - (dense * score).sum(-1, keepdim=True))
            if case["renormalize"]:   # the scores that were not chosen cancel
                dl = torch.where(torch.zeros_like(l).scatter_add_(1, e, has.float()) > 0, dl, 0.0)
        else:
            s = score.gather(1, e)
            dl = torch.zeros_like(l).scatter_add_(1, e, torch.where(has, g * s * (1 - s), 0.0))
        out["dlogits"] = dl.to(st["logits"].dtype)
    return out


def _plain_rows(st):
    case = st["case"]
    x, y, w = st["x"].detach().float(), st["y"].detach().float(), st["weights"].detach()
    p, token = st["places"].long(), st["order"].long() // case["top"]
    dt = st["x"].dtype
    out = {"xs": x[token].to(dt), "y": (y[p] * w[..., None]).sum(1).to(dt)}
    if case["train"]:
        dy = st["dy"].float()
        out["dx"] = st["dxs"].float()[p].sum(1).to(dt)
        out["dys"] = (dy[token] * w.flatten()[st["order"].long()][:, None]).to(dt)
        out["dw"] = (y[p] * dy[:, None]).sum(-1)
    return out


def _plain_adapters(st, x, y, a, b):
    """y + c B (A x), adapter by adapter; the sum A x too."""
    out, h = y.detach().float().clone(), torch.zeros((x.shape[0], a.shape[1]), device="cuda")
    for i in range(a.shape[0]):
        at = (st["ids"] == i).nonzero()[:, 0]
        h[at] = x.detach().float()[at] @ a[i].detach().float().T
        out[at] += st["scales"][i] * (h[at] @ b[i].detach().float().T)
    return out.to(y.dtype), h


def _plain_adapters_train(st):
    y, h = _plain_adapters(st, st["x"], st["y"], st["a"], st["b"])
    x, dy, a, b = (st[n].detach().float() for n in ("x", "dy", "a", "b"))
    dx, da, db = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    for i in range(a.shape[0]):
        at = (st["ids"] == i).nonzero()[:, 0]
        d = dy[at] * st["scales"][i]
        g = d @ b[i]
        dx[at], da[i], db[i] = g @ a[i], g.T @ x[at], d.T @ h[at]
    dt = st["x"].dtype
    return {"y": y, "d_y": st["dy"], "dx": dx.to(dt), "da": da.to(dt), "db": db.to(dt)}


def run(st):
    case = st["case"]
    kind, train = case["kind"], case["train"]
    if not own:
        if kind == "route":
            return _plain_route(st)
        if kind == "rows":
            return _plain_rows(st)
        if train:
            return _plain_adapters_train(st)
        return {"up": _plain_adapters(st, st["x"], st["y"], st["a"], st["b"])[0],
                "down": _plain_adapters(st, st["x2"], st["y2"], st["a2"], st["b2"])[0]}
    import mlx_b200 as mb
    from mlx_b200 import grad
    if kind == "route":
        args = dict(scoring=case["scoring"], bias=st["bias"], groups=case["groups"], top_groups=case["top_groups"],
                    group_best=case["group_best"], renormalize=case["renormalize"], scale=case["scale"])
        routing = (grad if train else mb).route_experts(st["logits"], case["top"], **args)
        out = {"weights": routing.weights.detach() if train else routing.weights, "experts": routing.experts, "sizes": routing.sizes,
               "places": routing.places, "order": routing.order}
        if train:
            out["dlogits"], = torch.autograd.grad(routing.weights, st["logits"], st["dw"])
        return out
    if kind == "rows":
        routing = mb.Routing(st["weights"], st["experts"], st["sizes"], st["places"], st["order"])
        if not train:
            return {"xs": mb.dispatch_rows(st["x"], routing), "y": mb.combine_rows(st["y"], routing)}
        xs, y = grad.dispatch_rows(st["x"], routing), grad.combine_rows(st["y"], routing)
        dx, dys, dw = torch.autograd.grad((xs, y), (st["x"], st["y"], st["weights"]), (st["dxs"], st["dy"]))
        return {"xs": xs.detach(), "y": y.detach(), "dx": dx, "dys": dys, "dw": dw}
    groups = mb.group_rows(st["ids"], case["L"])
    if not train:
        return {"up": mb.add_adapters(st["y"], st["x"], st["a"], st["b"], groups, st["scales"]),
                "down": mb.add_adapters(st["y2"], st["x2"], st["a2"], st["b2"], groups, st["scales"])}
    y = grad.add_adapters(st["y"], st["x"], st["a"], st["b"], groups, st["scales"])
    d_y, dx, da, db = torch.autograd.grad(y, (st["y"], st["x"], st["a"], st["b"]), st["dy"])
    return {"y": y.detach(), "d_y": d_y, "dx": dx, "da": da, "db": db}


# ------------------------------------------------------------------------------------------------ from the definitions, in 64 bits
def _first_best(key, count):
    """Indices of the `count` largest of every row, equal ones by index: each step takes the first element that equals the largest left."""
    key, picks = key.clone(), []
    taken = torch.zeros_like(key, dtype=torch.bool)
    for _ in range(count):
        left = torch.where(taken, -_INF, key)
        equal = (left == left.max(-1, keepdim=True).values) & ~taken
        pick = torch.where(equal, torch.arange(key.shape[1], device=key.device), key.shape[1]).min(-1).values
        taken.scatter_(1, pick[:, None], True)
        picks.append(pick)
    return torch.stack(picks, -1)


def _exact_route(case, st):
    E, G, top = case["E"], case["groups"], case["top"]
    l = st["logits"].detach().double().requires_grad_()
    logp = l - torch.logsumexp(l, -1, keepdim=True) if case["scoring"] == "softmax" else torch.nn.functional.logsigmoid(l)
    with torch.no_grad():
        score = logp.exp()
        key = l.detach().clone() if st["bias"] is None else score + st["bias"].double()
        if G > 1:
            member = key.reshape(-1, E // G)
            at = _first_best(member, case["group_best"])
            if case["group_best"] == 2 and st["bias"] is None:
                rank = score.reshape(-1, E // G).gather(1, at).sum(-1)
            else:
                rank = member.gather(1, at).sum(-1)
            kept = _first_best(rank.reshape(-1, G), case["top_groups"])
            off = torch.ones((key.shape[0], G), dtype=torch.bool, device=key.device).scatter_(1, kept, False)
            key = key.reshape(-1, G, E // G).masked_fill(off[..., None], -_INF).reshape(-1, E)
        experts = _first_best(key, top)
    chosen = logp.gather(1, experts)
    w = (torch.softmax(chosen, -1) if case["renormalize"] else chosen.exp()) * case["scale"]
    flat = experts.flatten()
    n = len(flat)
    order = (flat * n + torch.arange(n, device=flat.device)).sort().values % n
    places = torch.empty_like(order).scatter_(0, order, torch.arange(n, device=flat.device))
    sizes = (torch.searchsorted(flat[order], torch.arange(E + 1, device=flat.device))).diff()
    out = {"weights": w.detach(), "experts": experts.int(), "sizes": sizes.int(), "places": places.int().reshape(experts.shape), "order": order.int()}
    if case["train"]:
        out["dlogits"], = torch.autograd.grad(w, l, st["dw"].double())
    return out


def _exact_rows(case, st):
    T, top = case["T"], case["top"]
    y, w, p = st["y"].detach(), st["weights"].detach().double(), st["places"].long()
    out = {"xs": torch.zeros_like(y).double(), "y": 0}
    if case["train"]:
        dy = st["dy"].double()
        out.update(dx=0, dys=torch.zeros_like(y).double(), dw=torch.zeros_like(w))
    for j in range(top):
        out["xs"][p[:, j]] = st["x"].detach().double()
        out["y"] = out["y"] + w[:, j, None] * y[p[:, j]].double()
        if case["train"]:
            out["dx"] = out["dx"] + st["dxs"][p[:, j]].double()
            out["dys"][p[:, j]] = w[:, j, None] * dy
            out["dw"][:, j] = torch.einsum("td,td->t", dy, y[p[:, j]].double())
    return out


def _exact_adapters(st, x, y, a, b):
    x, a, b = x.detach().double(), a.detach(), b.detach()
    y = y.detach().double()
    for i in st["ids"].unique().tolist():
        if i >= 0:
            on = (st["ids"] == i).double()[:, None]
            if x.shape[0] > 64:
                rows = on[:, 0].nonzero()[:, 0]
                y[rows] = y[rows] + (x[rows] @ a[i].double().T * st["scales"][i].double()) @ b[i].double().T
            else:
                y = y + ((x * on) @ a[i].double().T * st["scales"][i].double()) @ b[i].double().T
    return y


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "route":
        return _exact_route(case, st)
    if case["kind"] == "rows":
        return _exact_rows(case, st)
    y = _exact_adapters(st, st["x"], st["y"], st["a"], st["b"])
    if not case["train"]:
        return {"up": y, "down": _exact_adapters(st, st["x2"], st["y2"], st["a2"], st["b2"])}
    x, dy = st["x"].detach().double(), st["dy"].double()
    dx, da, db = torch.zeros_like(x), torch.zeros(st["a"].shape, dtype=torch.float64, device="cuda"), torch.zeros(st["b"].shape, dtype=torch.float64, device="cuda")
    for i in range(case["L"]):
        rows = (st["ids"] == i).nonzero()[:, 0]
        c, ai, bi = st["scales"][i].double(), st["a"][i].detach().double(), st["b"][i].detach().double()
        back = torch.einsum("tn,nr->tr", dy[rows], bi)
        dx[rows] = c * torch.einsum("tr,rk->tk", back, ai)
        da[i] = c * torch.einsum("tr,tk->rk", back, x[rows])
        db[i] = c * torch.einsum("tn,tr->nr", dy[rows], torch.einsum("tk,rk->tr", x[rows], ai))
    return {"y": y, "d_y": dy, "dx": dx, "da": da, "db": db}
