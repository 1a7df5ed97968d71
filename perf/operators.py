"""Cases for the operators of image and video models: rotary positions with several axes, group norm with an
activation (channels last), and dropout whose mask is drawn again instead of stored.

`run` computes them in elementary torch operations, or, where `own` is true, through this package.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_handle = []


def _sideaware():
    """The loaded library, one handle for the process."""
    if not _handle:
        import l2_torch_alloc_b200
        _handle.append(l2_torch_alloc_b200.SideAware())
    return _handle[0]


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _rope(name, B, T, q, kv, head, axes, dtype, layout, arrangement, backward=False, theta=10000.0, far=0):
    return {"name": name, "op": "rope", "B": B, "T": T, "q": q, "kv": kv, "head": head, "axes": axes, "dtype": dtype,
            "layout": layout, "arrangement": arrangement, "backward": backward, "theta": theta, "far": far}


def _norm(name, N, S, C, G, dtype, silu=True, backward=False, params="fp32"):
    return {"name": name, "op": "norm", "N": N, "S": S, "C": C, "G": G, "dtype": dtype, "silu": silu,
            "backward": backward, "params": params}


def _drop(name, n, p, dtype, residual=False, backward=False):
    return {"name": name, "op": "dropout", "n": n, "p": p, "dtype": dtype, "residual": residual, "backward": backward}


def listed():
    return [
        # one new token for each of 64 running conversations about images, far into their contexts
        _rope("rope decode bf16", 64, 1, 32, 8, 128, "16,24,24", "bf16", "halves", "shared", theta=500000.0, far=100000),
        # a vision tower over four images: rows and columns, heads of 72
        _rope("rope image fp16", 4, 4097, 16, 16, 72, "18,18", "fp16", "halves", "own"),
        # a long video's tokens (time, height, width) through one layer of a video model
        _rope("rope video bf16", 1, 65536, 32, 8, 128, "22,21,21", "bf16", "interleaved", "own"),
        # gradient of the packed tensor, ragged length, heads of 96, axes dealt in turn
        _rope("rope backward fp32", 3, 1023, 12, 4, 96, "16,16,16", "fp32", "halves", "interleaved", backward=True, theta=1e6),
        # the innermost block of a denoiser, one image: latency
        _norm("norm 8x8x1280 bf16", 1, 64, 1280, 32, "bf16"),
        # the outermost blocks of a denoiser, a batch of eight
        _norm("norm 64x64x320 bf16", 8, 4096, 320, 32, "bf16", params="bf16"),
        # the last blocks of an image decoder
        _norm("norm 512x512x128 bf16", 2, 262144, 128, 32, "bf16"),
        # training of a middle block
        _norm("norm backward 32x32x640 fp16", 8, 1024, 640, 32, "fp16", backward=True),
        # odd picture sizes and groups of three channels, no activation
        _norm("norm backward 37x53x96 fp32", 3, 1961, 96, 32, "fp32", silu=False, backward=True),
        # one sequence of 64 tokens in front of its residual stream
        _drop("dropout 64x4096 bf16", 64 * 4096, 0.1, "bf16", residual=True),
        # a training batch of 4 sequences of 8192 tokens
        _drop("dropout 32768x4096 bf16", 32768 * 4096, 0.1, "bf16", residual=True),
        # gradient, odd element count
        _drop("dropout backward fp32", 10000019, 0.3, "fp32", backward=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("rope", "norm", "dropout"))
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    if op == "rope":
        head = rng.choice((32, 48, 64, 72, 80, 96, 128, 160, 256))
        q = rng.randint(1, 32)
        kv = rng.choice([k for k in (0, 1, 2, 4, 8, q) if k <= q])
        pairs = head // 2 if rng.random() < 0.75 else head // 4
        axes = rng.randint(1, 4)
        cuts = sorted(rng.sample(range(1, pairs), axes - 1))
        runs = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
        B = rng.choice((1, 1, 2, 3, 8, 33))
        most = 600e6 / (4 if dtype == "fp32" else 2) / ((q + 2 * kv) * head * B)
        T = max(1, _log(rng, 1, max(2, most)))
        c = _rope("", B, T, q, kv, head, ",".join(map(str, runs)), dtype, rng.choice(("halves", "interleaved")),
                  rng.choice(("own", "shared", "interleaved")), rng.random() < 0.4, rng.choice((100.0, 10000.0, 500000.0)),
                  rng.choice((0, 0, 1000, 1000000)))
    elif op == "norm":
        G = rng.choice((1, 2, 8, 16, 32, 32, 32))
        C = G * rng.choice((1, 2, 3, 4, 5, 8, 10, 16, 20, 30, 40))
        N = rng.choice((1, 1, 2, 3, 4, 8, 16))
        S = _log(rng, 1, max(2, 33e6 / (C * N)))
        c = _norm("", N, S, C, G, dtype, rng.random() < 0.7, rng.random() < 0.5, rng.choice(("fp32", dtype)))
    else:
        c = _drop("", _log(rng, 1, 60e6), rng.choice((0.05, 0.1, 0.2, 0.5, 0.9)), dtype, rng.random() < 0.5)
        if not c["residual"]:
            c["backward"] = rng.random() < 0.5
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _pairs(case):
    return [int(v) for v in case["axes"].split(",")]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    s = {"case": case}
    if case["op"] == "rope":
        B, T, heads = case["B"], case["T"], case["q"] + 2 * case["kv"]
        s["qkv"] = normal(B, T, heads, case["head"]).to(dtype)
        # a picture's or a video's grid: the first axis is the slowest, each axis has its own extent, every sequence its own start
        axes = len(_pairs(case))
        side = max(1, round(T ** (1.0 / axes)))
        t = torch.arange(T, device="cuda", dtype=torch.int64)
        rows = [(t // side ** (axes - 1 - a)) % (side if a else T + 1) for a in range(axes)]
        start = torch.randint(0, case["far"] + 1 if case["far"] else 8, (1, B, 1), device="cuda", generator=g)
        s["positions"] = (torch.stack(rows).unsqueeze(1) + start).to(torch.int32).contiguous()
        if own:
            s["spectrum"] = _sideaware().rope_axes_spectrum(_pairs(case), theta=case["theta"], arrangement=case["arrangement"])
    elif case["op"] == "norm":
        N, S, C, G = case["N"], case["S"], case["C"], case["G"]
        params = DTYPES[case["params"]]
        x = normal(N, S, C) * (0.5 + torch.rand(C, device="cuda", generator=g)) + 0.5 * normal(N, 1, C)
        s["x"] = x.to(dtype)
        s["weight"] = (1.0 + 0.2 * normal(C)).to(params)
        s["bias"] = (0.2 * normal(C)).to(params)
        s["out"] = torch.empty_like(s["x"])
        s["mean"] = torch.empty(N, G, device="cuda")
        s["rstd"] = torch.empty(N, G, device="cuda")
        if case["backward"]:
            s["dout"] = normal(N, S, C).to(dtype)
            s["dweight"], s["dbias"] = torch.empty_like(s["weight"]), torch.empty_like(s["bias"])
            grouped = s["x"].double().view(N, S, G, C // G)
            var, mean = torch.var_mean(grouped, dim=(1, 3), correction=0)
            s["mean"].copy_(mean)
            s["rstd"].copy_((var + 1e-5).rsqrt())
    else:
        s["x"] = normal(case["n"]).to(dtype)
        s["out"] = torch.empty_like(s["x"])
        s["residual"] = normal(case["n"]).to(dtype) if case["residual"] else None
        s["rng"] = torch.randint(0, 2 ** 62, (2,), device="cuda", generator=g)
    if own:
        _sideaware()
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if case["op"] == "rope":
        return _run_rope(case, s)
    if case["op"] == "norm":
        return _run_norm_backward(case, s) if case["backward"] else _run_norm(case, s)
    return _run_dropout(case, s)


def _frequencies(case):
    """Angle of each pair for one step of its axis, in 64 bits, and that axis."""
    runs = _pairs(case)
    total = sum(runs)
    if case["arrangement"] == "own":
        spots = [(a, j / n) for a, n in enumerate(runs) for j in range(n)]
    elif case["arrangement"] == "shared":
        spots = [(a, None) for a, n in enumerate(runs) for _ in range(n)]
    else:  # one pair for each axis in turn, as long as it has any left
        spots = [(a, None) for j in range(max(runs)) for a, n in enumerate(runs) if j < n]
    power = [i / total if p is None else p for i, (_, p) in enumerate(spots)]
    return [case["theta"] ** -p for p in power], [a for a, _ in spots]


def _run_rope(case, s):
    qkv, heads = s["qkv"], case["q"] + case["kv"]
    if own:
        call = _sideaware().rope_axes_backward if case["backward"] else _sideaware().rope_axes_forward
        call(qkv, s["positions"], s["spectrum"], case["q"], case["kv"], layout=case["layout"])
        return qkv
    if "frequency" not in s:  # a program's plan: kept with the state
        frequency, axis = _frequencies(case)
        s["frequency"] = torch.tensor(frequency, dtype=torch.float64, device="cuda")
        s["axis"] = torch.tensor(axis, device="cuda")
    angle = s["positions"].double()[s["axis"]].permute(1, 2, 0) * s["frequency"]  # [B, T, pairs]
    cos, sin = angle.cos().float().unsqueeze(2), angle.sin().float().unsqueeze(2)
    if case["backward"]:
        sin = -sin
    pairs = cos.shape[-1]
    x = qkv[:, :, :heads, :2 * pairs].float()
    if case["layout"] == "halves":
        a, b = x[..., :pairs], x[..., pairs:]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)
    else:
        a, b = x[..., 0::2], x[..., 1::2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    qkv[:, :, :heads, :2 * pairs] = turned.to(qkv.dtype)
    return qkv


def _run_norm(case, s):
    x, N, S, C, G = s["x"], case["N"], case["S"], case["C"], case["G"]
    if own:
        _sideaware().group_norm_forward(s["out"], s["mean"], s["rstd"], x, s["weight"], s["bias"], G, 1e-5, silu=case["silu"])
        return s["out"], s["mean"], s["rstd"]
    g = x.float().view(N, S, G, C // G)
    mean = g.mean(dim=(1, 3))
    centred = g - mean[:, None, :, None]
    rstd = 1.0 / ((centred * centred).mean(dim=(1, 3)) + 1e-5).sqrt()
    y = (centred * rstd[:, None, :, None]).view(N, S, C) * s["weight"].float() + s["bias"].float()
    if case["silu"]:
        y = y / (1.0 + (-y).exp())
    return y.to(x.dtype), mean, rstd


def _run_norm_backward(case, s):
    x, N, S, C, G = s["x"], case["N"], case["S"], case["C"], case["G"]
    if own:
        _sideaware().group_norm_backward(s["out"], s["dweight"], s["dbias"], s["dout"], x, s["mean"], s["rstd"], s["weight"],
                                         s["bias"], G, silu=case["silu"])
        return s["out"], s["dweight"], s["dbias"]
    weight, rstd = s["weight"].float(), s["rstd"][:, None, :, None]
    unit = ((x.float().view(N, S, G, C // G) - s["mean"][:, None, :, None]) * rstd).view(N, S, C)
    dy = s["dout"].float()
    if case["silu"]:
        z = unit * weight + s["bias"].float()
        sig = 1.0 / (1.0 + (-z).exp())
        dy = dy * (sig * (1.0 + z * (1.0 - sig)))
    dweight, dbias = (dy * unit).sum(dim=(0, 1)), dy.sum(dim=(0, 1))
    u = unit.view(N, S, G, C // G)
    d = (dy * weight).view(N, S, G, C // G)
    dx = rstd * (d - d.mean(dim=(1, 3), keepdim=True) - u * (d * u).mean(dim=(1, 3), keepdim=True))
    return dx.view(N, S, C).to(x.dtype), dweight.to(s["weight"].dtype), dbias.to(s["weight"].dtype)


M32 = 0xFFFFFFFF


def _philox(even, odd, key):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw, 2011) on 32-bit words held in int64: `even` holds words 0 and 2 of the
    counters, `odd` words 1 and 3, `key` the two halves of the key."""
    factor = torch.tensor([0xD2511F53, 0xCD9E8D57], device=key.device).view(2, 1, 1)
    keys = (key + torch.arange(10, device=key.device).view(10, 1) * torch.tensor([0x9E3779B9, 0xBB67AE85], device=key.device)) & M32
    for k in keys.view(10, 2, 1, 1):
        product = even * factor  # modulo 2^64: the upper halves are taken with a mask
        even, odd = ((product >> 32) & M32).flip(0) ^ odd ^ k, (product & M32).flip(0)
    return torch.stack((even[0], odd[0], even[1], odd[1]), dim=-1)


def _uniform32(n, rng):
    """The 32-bit random number of each of n elements: its upper half from the block of its eight elements, its lower half
    from the block at the same place of the other half of the counter's range."""
    group = torch.arange((n + 7) // 8, device=rng.device, dtype=torch.int64)
    word1 = (group >> 32) + torch.tensor([[0], [1 << 31]], device=rng.device)  # row 0: the upper halves' blocks, row 1: the lower halves'
    seed, call = torch.stack((rng & M32, (rng >> 32) & M32), dim=-1)
    even = torch.stack(((group & M32).expand(2, -1), call[0].expand_as(word1)))
    odd = torch.stack((word1, call[1].expand_as(word1)))
    words = _philox(even, odd, seed)
    upper, lower = torch.stack((words & 0xFFFF, words >> 16), dim=-1).view(2, -1)
    return ((upper << 16) | lower)[:n]


def _run_dropout(case, s):
    x, p = s["x"], case["p"]
    if own:
        if case["backward"]:
            _sideaware().dropout_backward(s["out"], x, s["rng"], p)
        else:
            _sideaware().dropout_forward(s["out"], x, s["rng"], p, residual=s["residual"])
        return s["out"]
    keep = _uniform32(x.numel(), s["rng"]) >= round(p * 2 ** 32)
    y = torch.where(keep, x.float() * (1.0 / (1.0 - p)), 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(x.dtype)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rope":
        tokens, pairs = case["B"] * case["T"], sum(_pairs(case))
        turned = tokens * (case["q"] + case["kv"]) * pairs  # value heads and the part that is not turned stay where they are
        return {"bytes": 4 * turned * e + 4 * tokens * len(_pairs(case)), "flops": 6 * turned}
    if case["op"] == "norm":
        n = case["N"] * case["S"] * case["C"]
        p = case["C"] * (4 if case["params"] == "fp32" else 2)
        stats = 8 * case["N"] * case["G"]
        if case["backward"]:
            return {"bytes": 3 * n * e + 4 * p + stats, "flops": (24 if case["silu"] else 12) * n}
        return {"bytes": 2 * n * e + 2 * p + stats, "flops": (12 if case["silu"] else 7) * n}
    return {"bytes": case["n"] * e * (3 if case["residual"] else 2) + 16, "flops": 3 * case["n"]}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "rope":
        return _exact_rope(case, s)
    if case["op"] == "norm":
        return _exact_norm(case, s)
    return _exact_dropout(case, s)


def _exact_rope(case, s):
    """Each pair as a complex number, times e^(i angle); one sequence and a few thousand tokens at a time."""
    runs, theta = _pairs(case), case["theta"]
    axis, power, left = [], [], list(runs)
    a = 0
    for i in range(sum(runs)):
        if case["arrangement"] == "interleaved":
            while not left[a % len(runs)]:
                a += 1
        else:
            a = next(k for k in range(len(runs)) if left[k])
        k = a % len(runs)
        power.append((runs[k] - left[k]) / runs[k] if case["arrangement"] == "own" else i / sum(runs))
        axis.append(k)
        left[k] -= 1
        a += case["arrangement"] == "interleaved"
    pairs, heads = len(axis), case["q"] + case["kv"]
    step = torch.exp(torch.tensor(power, dtype=torch.float64, device="cuda") * -math.log(theta))
    out = s["qkv"].double()
    sign = -1.0 if case["backward"] else 1.0
    for b in range(case["B"]):
        for t0 in range(0, case["T"], 8192):
            place = s["positions"][axis, b, t0:t0 + 8192].double().T
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda").expand(place.shape).contiguous(), sign * place * step)
            part = out[b, t0:t0 + 8192, :heads, :2 * pairs]
            if case["layout"] == "halves":
                z = torch.complex(part[..., :pairs], part[..., pairs:]) * turn[:, None]
                part.copy_(torch.cat((z.real, z.imag), dim=-1))
            else:
                z = torch.complex(part[..., 0::2], part[..., 1::2]) * turn[:, None]
                part.copy_(torch.view_as_real(z).flatten(-2))
    return out


def _exact_norm(case, s):
    """Group norm as a function of 64-bit leaves; the gradients by reverse differentiation of the definition."""
    N, S, C, G = case["N"], case["S"], case["C"], case["G"]
    x, w, b = (s[k].double() for k in ("x", "weight", "bias"))
    if case["backward"]:
        x, w, b = (v.requires_grad_() for v in (x, w, b))
    rows = x.view(N, S, G, C // G).permute(0, 2, 1, 3).reshape(N, G, -1)
    mean = rows.sum(-1) / rows.shape[-1]
    var = (rows - mean.unsqueeze(-1)).pow(2).sum(-1) / rows.shape[-1]
    rstd = (var + 1e-5).pow(-0.5)
    unit = ((rows - mean.unsqueeze(-1)) * rstd.unsqueeze(-1)).view(N, G, S, C // G).permute(0, 2, 1, 3).reshape(N, S, C)
    y = unit * w + b
    if case["silu"]:
        y = y * torch.sigmoid(y)
    if not case["backward"]:
        return y, mean, rstd
    return torch.autograd.grad(y, (x, w, b), s["dout"].double())


def _exact_dropout(case, s):
    """The generator again, its products put together from 16-bit pieces."""
    n, rng, p = case["n"], s["rng"].tolist(), case["p"]
    group = torch.arange((n + 7) // 8, device="cuda", dtype=torch.int64)

    def product(c, m):
        low, high = c & 0xFFFF, c >> 16
        mid = high * (m & 0xFFFF) + (low * (m & 0xFFFF) >> 16)
        cross = low * (m >> 16) + (mid & 0xFFFF)
        return high * (m >> 16) + (mid >> 16) + (cross >> 16), ((cross & 0xFFFF) << 16) | (low * (m & 0xFFFF) & 0xFFFF)

    def block(second):
        x = [group % 2 ** 32, group // 2 ** 32 + second * 2 ** 31, torch.full_like(group, rng[1] % 2 ** 32), torch.full_like(group, rng[1] >> 32)]
        for r in range(10):
            h0, l0 = product(x[0], 0xD2511F53)
            h1, l1 = product(x[2], 0xCD9E8D57)
            x = [h1 ^ x[1] ^ ((rng[0] + r * 0x9E3779B9) % 2 ** 32), l1, h0 ^ x[3] ^ (((rng[0] >> 32) + r * 0xBB67AE85) % 2 ** 32), l0]
        return x

    u = torch.empty(8, group.numel(), dtype=torch.int64, device="cuda")
    for word, (a, b) in enumerate(zip(block(0), block(1))):
        u[2 * word] = (a % 65536) * 65536 + b % 65536
        u[2 * word + 1] = (a // 65536) * 65536 + b // 65536
    kept = u.T.reshape(-1)[:n] >= int(round(p * 4294967296.0))
    y = s["x"].double() / (1.0 - p) * kept
    return y if s["residual"] is None else y + s["residual"].double()
