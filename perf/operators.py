"""Microscaled 4-bit products and products grouped by expert, as cases that a timing harness can run.

`kind` of a case says which operators it goes through:

    convert       quantize and dequantize of a matrix in a microscaled 4-bit mode: a checkpoint being converted and checked
    qqmm          qqmm: M rows of activations, quantised on the way, through one linear layer of 4-bit weights
    experts       grouped_mm: rows sorted by expert through one 16-bit projection of a mixture-of-experts layer
    train         grad.grouped_mm and its backward pass: the same projection being trained (y, dx and dw)
    experts4      grouped_qqmm: the projection with 4-bit weights

`own` says who computes: the framework's operators, or (False) their plain forms below, which follow the formulas in
32 bits and round once at the end.

E2M1, the 4-bit type: sign, two exponent bits, one mantissa bit; magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6.
mxfp4: groups of 32 values share the power of two 2^(floor(log2 amax) - 2).
nvfp4: groups of 16 share an E4M3 number, amax / (6 G) rounded; G is one fp32 number per tensor.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_GROUP = {"mxfp4": 32, "nvfp4": 16}
_E, _K, _N = 8, 4096, 14336   # the experts and widths of this repository's mixture-of-experts benchmark


def _convert(N, K, mode, dtype):
    return {"kind": "convert", "N": N, "K": K, "mode": mode, "dtype": dtype}


def _qqmm(M, N, K, mode, dtype):
    return {"kind": "qqmm", "M": M, "N": N, "K": K, "mode": mode, "dtype": dtype}


def _experts(kind, tokens, E, top, N, K, dtype, mode="", transpose=True):
    return {"kind": kind, "tokens": tokens, "E": E, "top": top, "N": N, "K": K, "dtype": dtype, "mode": mode, "transpose": transpose}


def listed():
    return [
        # the widest matrix of a checkpoint
        {"name": "convert mxfp4", **_convert(28672, 8192, "mxfp4", "bf16")},
        # a small half-precision matrix with an odd number of rows, in the mode with a scale for the whole tensor
        {"name": "convert nvfp4 odd", **_convert(1531, 2064, "nvfp4", "f16")},
        # one token through a square attention projection: the smallest call of a decode loop
        {"name": "qqmm 1 row", **_qqmm(1, 4096, 4096, "nvfp4", "bf16")},
        # sixteen sequences decoded together through an MLP up-projection
        {"name": "qqmm 16 rows", **_qqmm(16, _N, _K, "mxfp4", "bf16")},
        # a server's batch through a down-projection: neither decode nor a full tile, half precision
        {"name": "qqmm 57 rows f16", **_qqmm(57, 4096, 11008, "mxfp4", "f16")},
        # a long prompt: the dense tensor-core case
        {"name": "qqmm 4096 rows", **_qqmm(4096, _N, _K, "nvfp4", "bf16")},
        # four sequences decoded together, top-2 of 8 experts: a row or two per expert, some experts without any
        {"name": "experts 4 tokens", **_experts("experts", 4, _E, 2, _N, _K, "bf16")},
        # a prompt through the same projection
        {"name": "experts 512 tokens", **_experts("experts", 512, _E, 2, _N, _K, "bf16")},
        # the projection being trained
        {"name": "train 2048 tokens", **_experts("train", 2048, _E, 2, _N, _K, "bf16")},
        # many narrow experts, half precision, an odd number of tokens, weights stored the other way round
        {"name": "train 1531 tokens f16", **_experts("train", 1531, 32, 4, 1536, 2048, "f16", transpose=False)},
        # decoding with 4-bit experts
        {"name": "experts4 4 tokens", **_experts("experts4", 4, _E, 2, _N, _K, "bf16", "mxfp4")},
        # a prompt through them
        {"name": "experts4 512 tokens", **_experts("experts4", 512, _E, 2, _N, _K, "bf16", "nvfp4")},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges: rows from one to the largest listed, widths that are mostly whole 64s, sometimes any
    whole number of 4-bit groups (16 bits: any number), every mode and type, both layouts of the weights, 2 to 64 experts
    that together are no larger than the listed ones."""
    most = {key: max(work(c)[key] for c in listed()) for key in ("bytes", "flops")}
    while True:
        kind = rng.choice(["convert", "qqmm", "qqmm", "experts", "train", "experts4"])
        mode = rng.choice(["mxfp4", "nvfp4"])
        g = _GROUP[mode]
        dtype = rng.choice(["bf16", "bf16", "f16"])
        N, K = _log_int(rng, 512, 14336), _log_int(rng, 512, 14336)
        odd = rng.random() < 0.25
        if not odd:
            N, K = N // 64 * 64, K // 64 * 64
        elif kind in ("convert", "qqmm", "experts4"):
            K = K // g * g
        if kind == "convert":
            c = _convert(_log_int(rng, 64, 28672), K, mode, rng.choice(["bf16", "f16", "f32"]))
        elif kind == "qqmm":
            c = _qqmm(_log_int(rng, 1, 4096), N, K, mode, dtype)
        else:
            E = _log_int(rng, 2, 64)
            top = rng.randint(1, min(E, 8))
            tokens = _log_int(rng, 1, 4096)
            if E * N * K > _E * _N * _K:
                continue
            if kind == "experts4":
                c = _experts(kind, tokens, E, top, N, K, dtype, mode)
            else:
                c = _experts(kind, tokens, E, top, N, K, dtype, transpose=rng.random() < 0.6)
        if all(work(c)[key] <= most[key] for key in most):
            return c


def work(case):
    """Bytes that have to be read and written once, and operations."""
    b = 4 if case["dtype"] == "f32" else 2
    N, K = case["N"], case["K"]
    if case["kind"] == "convert":
        packed = N * K // 2 + N * K // _GROUP[case["mode"]]
        return {"bytes": 2 * (N * K * b + packed), "flops": 2 * N * K}
    if case["kind"] == "qqmm":
        M = case["M"]
        return {"bytes": M * K * b + N * K // 2 + N * K // _GROUP[case["mode"]] + M * N * b, "flops": 2 * M * N * K}
    rows = case["tokens"] * case["top"]
    used = min(case["E"], rows)   # experts that can have rows
    act, flops = (rows * K + rows * N) * b, 2 * rows * N * K
    if case["kind"] == "experts4":
        return {"bytes": used * (N * K // 2 + N * K // _GROUP[case["mode"]]) + act, "flops": flops}
    if case["kind"] == "experts":
        return {"bytes": used * N * K * b + act, "flops": flops}
    # forward as above; backward reads dy, x and the weights again and writes dx and every expert's dw
    return {"bytes": 2 * used * N * K * b + case["E"] * N * K * b + 2 * act + act, "flops": 3 * flops}


# ------------------------------------------------------------------------------------------------ the 4-bit modes, plainly
def _e2m1(t):
    """Codes of |t| (0..7): nearest, ties to the even code."""
    c = torch.zeros_like(t, dtype=torch.uint8)
    c += t > 0.25
    c += t >= 0.75
    c += t > 1.25
    c += t >= 1.75
    c += t > 2.5
    c += t >= 3.5
    c += t > 5.0
    return c


def _quantize(w, mode, G):
    """fp32 w [rows, K] -> (codes uint8 [rows, K], scale codes uint8 [rows, K/g])."""
    g = _GROUP[mode]
    v = w.unflatten(-1, (-1, g))
    amax = v.abs().amax(-1)
    if mode == "mxfp4":
        e = ((amax.view(torch.int32) >> 23) - 2).clamp_min(0)   # the exponent's field: floor(log2) + 127
        d = torch.exp2((e - 127).float())
        s = e.to(torch.uint8)
    else:
        six = 6.0 * G
        s8 = (amax / six).clamp_max(448.0).to(torch.float8_e4m3fn)
        d = s8.float() * G
        s = s8.view(torch.uint8)
    t = torch.where((d == 0)[..., None], 0.0, v.abs() / d[..., None])
    c = _e2m1(t) + torch.signbit(v).to(torch.uint8) * 8
    return c.flatten(-2), s


def _pack(c):
    return (c[..., 0::2] | (c[..., 1::2] << 4)).contiguous().view(torch.uint32)


def _scale_values(s, mode):
    return torch.exp2(s.float() - 127) if mode == "mxfp4" else s.view(torch.float8_e4m3fn).float()


def _values(wq, s, mode):
    """fp32 values of packed codes and scales, without the tensor's own scale."""
    b = wq.view(torch.uint8)
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=b.device)
    v = torch.stack((table[(b & 15).int()], table[(b >> 4).int()]), -1).flatten(-2)
    return (v.unflatten(-1, (-1, _GROUP[mode])) * _scale_values(s, mode)[..., None]).flatten(-2)


# ------------------------------------------------------------------------------------------------ inputs
def _routing(case, gen):
    """Rows per expert: every token takes `top` different experts, some of which are asked for more often than others."""
    E = case["E"]
    p = torch.rand(E, generator=gen) + 0.25
    picks = torch.multinomial(p.expand(case["tokens"], E), case["top"], generator=gen)
    return torch.bincount(picks.flatten(), minlength=E)


def _global_scale(t):
    """The usual choice: the largest value of the tensor becomes the largest scale times the largest code."""
    return (t.abs().amax().float() / (448.0 * 6.0)).reshape(1)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dt, N, K = _DTYPES[case["dtype"]], case["N"], case["K"]

    def normal(shape, std, dtype=dt):
        return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)

    st = {"case": case}
    if case["kind"] == "convert":
        st["w"] = normal((N, K), 0.02)
        st["G"] = _global_scale(st["w"]) if case["mode"] == "nvfp4" else None
        return st
    if case["kind"] == "qqmm":
        st["x"] = normal((case["M"], K), 1.0)
        shape = (N, K)
    else:
        sizes = _routing(case, torch.Generator().manual_seed(seed))
        rows = case["tokens"] * case["top"]
        st["most"] = int(sizes.max())
        st["sizes"] = sizes.cuda()
        st["x"] = normal((rows, K), 1.0)
        shape = (case["E"], N, K) if case["transpose"] else (case["E"], K, N)
    w = normal(shape, 0.02)
    if case["kind"] in ("experts", "train"):
        st["w"] = w
        if case["kind"] == "train":
            st["dy"] = normal((st["x"].shape[0], N), 0.01)
            st["x"].requires_grad_()
            st["w"].requires_grad_()
        return st
    # 4-bit weights as a checkpoint holds them; the activations' scale is known from calibration
    st["Gw"] = _global_scale(w) if case["mode"] == "nvfp4" else None
    st["Gx"] = _global_scale(st["x"]) if case["mode"] == "nvfp4" else None
    c, s = _quantize(w.float().reshape(-1, K), case["mode"], st["Gw"])
    st["wq"], st["scales"] = _pack(c).reshape(*shape[:-1], -1), s.reshape(*shape[:-1], -1)
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _rows(st):
    """Of every row of x: its expert, and its place among the expert's rows; of every place (expert, i): its row, and whether it has one."""
    sizes, T, dev = st["sizes"], st["x"].shape[0], st["sizes"].device
    E = sizes.shape[0]
    first = sizes.cumsum(0) - sizes
    e = torch.repeat_interleave(torch.arange(E, device=dev), sizes, output_size=T)
    i = torch.arange(T, device=dev) - first[e]
    at = first[:, None] + torch.arange(st["most"], device=dev)
    has = torch.arange(st["most"], device=dev) < sizes[:, None]
    return e, i, at.clamp_max(T - 1), has


def _spread(t, at, has):
    return torch.where(has[..., None], t.detach().float()[at], 0.0)   # [E, most, columns]


def _plain(st):
    case = st["case"]
    kind, mode = case["kind"], case["mode"] if "mode" in case else ""
    if kind == "convert":
        w = st["w"].float()
        c, s = _quantize(w, mode, st["G"])
        v = _values(_pack(c), s, mode)
        return {"values": (v if st["G"] is None else v * st["G"]).to(st["w"].dtype), "scales": _scale_values(s, mode)}
    x = st["x"]
    if kind in ("qqmm", "experts4"):
        c, s = _quantize(x.float(), mode, st["Gx"])
        xv, wv = _values(_pack(c), s, mode), _values(st["wq"], st["scales"], mode)
        if kind == "qqmm":
            y = xv @ wv.T
        else:
            e, i, at, has = _rows(st)
            y = torch.bmm(_spread(xv, at, has), wv.transpose(1, 2))[e, i]
        if mode == "nvfp4":
            y = y * (st["Gx"] * st["Gw"])
        return {"y": y.to(x.dtype)}
    e, i, at, has = _rows(st)
    w = st["w"].detach().float()
    if not case["transpose"]:
        w = w.transpose(1, 2)
    xs = _spread(x, at, has)
    y = torch.bmm(xs, w.transpose(1, 2))[e, i].to(x.dtype)
    if kind == "experts":
        return {"y": y}
    dys = _spread(st["dy"], at, has)
    dx = torch.bmm(dys, w)[e, i].to(x.dtype)
    dw = torch.bmm(dys.transpose(1, 2), xs) if case["transpose"] else torch.bmm(xs.transpose(1, 2), dys)
    return {"y": y, "dx": dx, "dw": dw.to(x.dtype)}


def run(st):
    if not own:
        return _plain(st)
    import mlx_b200
    case = st["case"]
    kind = case["kind"]
    if kind == "convert":
        mode = case["mode"]
        wq, s = mlx_b200.quantize(st["w"], mode=mode, global_scale=st["G"])
        v = mlx_b200.dequantize(wq, s, mode=mode, global_scale=st["G"], dtype=st["w"].dtype)
        return {"values": v, "scales": _scale_values(s, mode)}
    if kind == "qqmm":
        return {"y": mlx_b200.qqmm(st["x"], st["wq"], st["scales"], mode=case["mode"], global_scale_x=st["Gx"], global_scale_w=st["Gw"])}
    if kind == "experts4":
        return {"y": mlx_b200.grouped_qqmm(st["x"], st["wq"], st["scales"], st["sizes"], mode=case["mode"],
                                           global_scale_x=st["Gx"], global_scale_w=st["Gw"])}
    if kind == "experts":
        return {"y": mlx_b200.grouped_mm(st["x"], st["w"], st["sizes"], case["transpose"])}
    from mlx_b200 import grad
    y = grad.grouped_mm(st["x"], st["w"], st["sizes"], case["transpose"])
    dx, dw = torch.autograd.grad(y, (st["x"], st["w"]), st["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw}


# ------------------------------------------------------------------------------------------------ from the definitions, in 64 bits
def _nearest(t, grid, even):
    """Values of `grid` (ascending, fp64) nearest to t >= 0; halfway: the one whose index is even (or its neighbour's is not)."""
    mid = (grid[1:] + grid[:-1]) / 2
    up = torch.searchsorted(mid, t, right=True)     # t at a midpoint: the upper one
    down = torch.searchsorted(mid, t, right=False)  # the lower one
    return grid[torch.where(up % 2 == even, up, down)]


def _exact_quantized(w, mode, G):
    """fp64: the values (without G) that w's codes and scales stand for, and the scales."""
    dev = w.device
    four = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=dev)
    v = w.double().reshape(w.shape[0], -1, _GROUP[mode])
    amax = v.abs().max(-1).values
    if mode == "mxfp4":
        _, e = torch.frexp(amax)                     # amax = m 2^e, m in [1/2, 1)
        e = torch.where(amax > 0, e - 3, -127).clamp(-127, 127)
        s = torch.ldexp(torch.ones_like(amax), e)
        d = s
    else:
        # E4M3: 8 subnormals in steps of 2^-9, then 8 numbers per octave up to 448
        g8 = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 9) for e in range(15) for m in range(8)]
        g8 = torch.tensor(g8[:-1], dtype=torch.float64, device=dev)
        s = _nearest((amax / (6 * G.double())).clamp(max=448.0), g8, 0)
        d = s * G.double()
    t = torch.where(d[..., None] > 0, v.abs() / d[..., None].clamp(min=1e-300), 0.0)
    q = _nearest(t, four, 0) * torch.sign(v)
    return (q * s[..., None]).reshape(w.shape), s


def _exact_stored(st):
    """fp64 values of the packed weights, without their global scale."""
    mode = st["case"]["mode"]
    words = st["wq"].view(torch.int32)
    nib = torch.stack([(words >> (4 * j)) & 15 for j in range(8)], -1).flatten(-2)
    m, e = (nib & 1).double(), (nib >> 1) & 3
    mag = torch.where(e == 0, 0.5 * m, torch.ldexp(1 + 0.5 * m, e - 1))
    mag = torch.where(nib >= 8, -mag, mag)
    c = st["scales"].int()
    if mode == "mxfp4":
        s = torch.ldexp(torch.ones(c.shape, dtype=torch.float64, device=c.device), c - 127)
    else:
        s = torch.where(c < 8, c.double() * 2.0 ** -9, torch.ldexp((8 + (c & 7)).double(), (c >> 3) - 10))
    return (mag.unflatten(-1, (-1, _GROUP[mode])) * s[..., None]).flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "convert":
        # rows in blocks: the searches work in 64-bit indexes
        vs, ss = zip(*(_exact_quantized(b, case["mode"], st["G"]) for b in st["w"].split(4096)))
        v = torch.cat(vs)
        return {"values": v if st["G"] is None else v * st["G"].double(), "scales": torch.cat(ss)}
    bounds = [0] + st["sizes"].cumsum(0).tolist() if "sizes" in st else None
    if kind in ("qqmm", "experts4"):
        x, _ = _exact_quantized(st["x"], case["mode"], st["Gx"])
        w = _exact_stored(st)
        if kind == "qqmm":
            y = x @ w.T
        else:
            y = torch.cat([x[a:b] @ w[e].T for e, (a, b) in enumerate(zip(bounds, bounds[1:]))])
        return {"y": y if st["Gx"] is None else y * (st["Gx"].double() * st["Gw"].double())}
    x, w = st["x"].detach().double(), st["w"].detach()
    y, dx, dw = [], [], []
    for e, (a, b) in enumerate(zip(bounds, bounds[1:])):
        we = w[e].double().T if case["transpose"] else w[e].double()    # [K, N]
        y.append(x[a:b] @ we)
        if kind == "train":
            dy = st["dy"][a:b].double()
            dx.append(dy @ we.T)
            dw.append(dy.T @ x[a:b] if case["transpose"] else x[a:b].T @ dy)
    if kind == "experts":
        return {"y": torch.cat(y)}
    return {"y": torch.cat(y), "dx": torch.cat(dx), "dw": torch.stack(dw)}
