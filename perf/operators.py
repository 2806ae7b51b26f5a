"""The layer and optimiser operators of wide networks as measurable cases: layer norm, the 8-bit product with a scale per block of
128, and the AdamW step over many tensors.

`run` computes a case either from elementary torch operations (own = False) or through nerf_amd's entry points (own = True), on the
inputs `prepare` made; `exact` is the same from the definitions in 64 bits.
"""
import math

import torch

own = False

BLOCK = 128          # values that share a scale, in 8-bit products and 8-bit states alike
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # one query's hidden vector in serving: a single row, where only latency counts
        {"name": "norm, one row", "op": "norm", "n": 1, "c": 4096, "type": "bfloat16", "train": False, "pad": 0},
        # the points of a training batch (1024 rays of 64 samples) at the framework's own width
        {"name": "norm, a ray batch's points", "op": "norm", "n": 65536, "c": 256, "type": "float32", "train": True, "pad": 0},
        # wide hidden layers in 16 bits
        {"name": "norm, wide rows", "op": "norm", "n": 8192, "c": 4096, "type": "bfloat16", "train": True, "pad": 0},
        # odd sizes, and rows that are a slice of a wider buffer (a skip connection's concatenation)
        {"name": "norm, odd strided rows", "op": "norm", "n": 10007, "c": 1537, "type": "float16", "train": True, "pad": 63},
        # a few queries through a wide layer whose weights are held in 8 bits: reading the weights bounds it
        {"name": "product, few rows", "op": "product", "m": 4, "k": 8192, "n": 8192, "type": "bfloat16", "train": False, "bias": True, "relu": True},
        # the points of a training batch through a hidden layer of the framework's own width, all in fp32
        {"name": "product, a ray batch's points", "op": "product", "m": 65536, "k": 256, "n": 256, "type": "float32", "train": True, "bias": True, "relu": False},
        # odd everywhere: a last block of 77 values, no dimension a multiple of a tile
        {"name": "product, odd sizes", "op": "product", "m": 1001, "k": 333, "n": 777, "type": "float16", "train": True, "bias": True, "relu": False},
        # rendering through a wide layer, weights held in 8 bits
        {"name": "product, wide layer", "op": "product", "m": 16384, "k": 4096, "n": 8192, "type": "bfloat16", "train": False, "bias": True, "relu": True},
        # one layer's share of a training step of a wide network
        {"name": "product, wide layer's training", "op": "product", "m": 8192, "k": 4096, "n": 4096, "type": "bfloat16", "train": True, "bias": True, "relu": False},
        # the update of two networks of the framework's own shape as 48 separate tensors: launch latency
        {"name": "update, two small networks", "op": "update", "width": 256, "depth": 8, "copies": 2, "type": "float32", "bits": 32},
        # wide networks in fp32 with states in 8 bits, odd width: tensors end inside a block of states
        {"name": "update, odd width in 8 bits", "op": "update", "width": 2047, "depth": 8, "copies": 2, "type": "float32", "bits": 8},
        # a large network in 16 bits with states in 32
        {"name": "update, large in 16 bits", "op": "update", "width": 4096, "depth": 8, "copies": 2, "type": "bfloat16", "bits": 32},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "product", "update"])
    kind = rng.choice(sorted(TYPES))
    if op == "norm":
        c = _log_int(rng, 8, 16384)
        return {"op": op, "n": _log_int(rng, 1, min(200000, 33554432 // c)), "c": c, "type": kind, "train": rng.random() < 0.7,
                "pad": rng.choice([0, 0, rng.randrange(1, 100)])}
    if op == "product":
        train = rng.random() < 0.5
        k, n = _log_int(rng, 16, 8192), _log_int(rng, 16, 8192)
        return {"op": op, "m": _log_int(rng, 1, min(100000, max(1, (1 << 36) // (k * n)))), "k": k, "n": n, "type": kind, "train": train,
                "bias": rng.random() < 0.7, "relu": (not train) and rng.random() < 0.5}
    return {"op": op, "width": _log_int(rng, 16, 4096), "depth": rng.randrange(1, 9), "copies": rng.randrange(1, 3), "type": kind,
            "bits": rng.choice([8, 32])}


def _shapes(case):
    """The parameter tensors of `copies` stacks of `depth` square layers (weight, bias, norm weight) and a 4-wide head."""
    w, d = case["width"], case["depth"]
    return ([(w, w), (w,), (w,)] * (d - 1) + [(w, 90), (w,), (4, w)]) * case["copies"]


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def prepare(case, seed):
    dev = _device()
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    dtype = TYPES[case["type"]]
    state = {"case": case}
    if case["op"] == "norm":
        n, c = case["n"], case["c"]
        wide = (normal(n, c + case["pad"]) * 1.5 + normal(n, 1)).to(dtype)    # every row with an offset of its own
        state["x"] = wide[:, :c]
        state["w"] = (1.0 + 0.2 * normal(c)).to(dtype)
        state["b"] = (0.1 * normal(c)).to(dtype)
        if case["train"]:
            state["dy"] = normal(n, c).to(dtype)
    elif case["op"] == "product":
        m, k, n = case["m"], case["k"], case["n"]
        # activations whose size differs from row to row and channel to channel, weights of a usual initialisation
        state["x"] = (normal(m, k) * torch.exp(0.5 * normal(m, 1)) * torch.exp(0.5 * normal(1, k))).to(dtype)
        w = (normal(n, k) / math.sqrt(k)).to(dtype)
        if case["bias"]:
            state["bias"] = (0.1 * normal(n)).to(dtype)
        if case["train"]:
            state["w"] = w
            state["dy"] = (normal(m, n) * 1e-3 * torch.exp(normal(m, 1))).to(dtype)
        else:                     # a program that only evaluates holds its weights in 8 bits
            state["codes"], state["scales"] = _quantize(w)
    else:
        # all tensors of a case lie in one arena, each from a multiple of 512 bytes on, as an allocator would place them
        shapes = _shapes(case)
        counts = [math.prod(s) for s in shapes]
        unit = 256                # elements; 512 bytes of the smallest type
        padded = [-(-c // unit) * unit for c in counts]
        starts = [sum(padded[:i]) for i in range(len(padded))]
        total = sum(padded)
        idx = torch.arange(total, device=dev) - torch.repeat_interleave(torch.tensor(starts, device=dev), torch.tensor(padded, device=dev))
        live = idx < torch.repeat_interleave(torch.tensor(counts, device=dev), torch.tensor(padded, device=dev))
        size = torch.exp(0.7 * normal(total // unit, 1)).expand(-1, unit).reshape(-1)      # gradients of different sizes
        master = normal(total) * 0.05 * live
        grad = normal(total) * 1e-3 * size * live
        m = normal(total) * 3e-4 * size * live
        v = (1e-3 * size) ** 2 * torch.exp(0.5 * normal(total)) * live
        state.update(shapes=shapes, counts=counts, starts=starts, padded=padded, step=99, p=master.to(dtype), g=grad.to(dtype))
        if dtype != torch.float32:
            state["master"] = state["p"].float() * (1 + 1e-3 * torch.rand(total, device=dev, generator=gen))
            state["p"] = state["master"].to(dtype)
        if case["bits"] == 32:
            state["m"], state["v"] = m, v
        else:
            mb, vb = m.view(-1, BLOCK), v.view(-1, BLOCK)
            sm, sv = mb.abs().amax(1, keepdim=True) / 448, vb.amax(1, keepdim=True) / 57344
            state["scale"] = torch.cat([sm, sv], 1)
            state["m"] = (mb / sm.clamp_min(1e-38)).clamp(-448, 448).to(torch.float8_e4m3fn).view(-1)
            state["v"] = (vb / sv.clamp_min(1e-38)).clamp(0, 57344).to(torch.float8_e5m2).view(-1)
    return state


# ------------------------------------------------------------------------------------------------
# the plain forms
# ------------------------------------------------------------------------------------------------
def _power(e):
    """2^e for whole e in [-126, 127], from its bits (a power function rounds)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantize(x):
    """Rows [r, k] -> e4m3 codes [r, k padded to a multiple of 128] and one power-of-two scale per row and 128 values as the exponent
    plus 127 [r, number of blocks padded to a multiple of 4]: the smallest power that takes the block's largest value to at most 448."""
    r, k = x.shape
    blocks = -(-k // BLOCK)
    wide = torch.zeros(r, blocks * BLOCK, device=x.device)
    wide[:, :k] = x
    wide = wide.view(r, blocks, BLOCK)
    frac, ex = torch.frexp(wide.abs().amax(2))                  # amax = frac 2^ex, 1/2 <= frac < 1; 448 = 0.875 * 2^9
    e = (ex - 9 + (frac > 0.875).int()).clamp_min(-126)
    codes = (wide * _power(-e)[:, :, None]).to(torch.float8_e4m3fn).view(r, blocks * BLOCK)
    scales = torch.zeros(r, -(-blocks // 4) * 4, device=x.device, dtype=torch.uint8)
    scales[:, :blocks] = (e + 127).to(torch.uint8)
    return codes, scales


def _dequantize(codes, scales, k):
    r, kp = codes.shape
    values = codes.float().view(r, kp // BLOCK, BLOCK)
    return (values * _power(scales[:, : kp // BLOCK].int() - 127)[:, :, None]).view(r, kp)[:, :k]


def _rounded(x):
    return _dequantize(*_quantize(x.float()), x.shape[1])


def _plain_norm(s):
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    dtype = s["x"].dtype
    mean = x.mean(1, keepdim=True)
    d = x - mean
    r = torch.rsqrt((d * d).mean(1, keepdim=True) + 1e-5)
    xh = d * r
    y = (xh * w + b).to(dtype)
    if "dy" not in s:
        return {"y": y}
    dy = s["dy"].float()
    g = dy * w
    dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(dtype), "dw": (dy * xh).sum(0).to(dtype), "db": dy.sum(0).to(dtype)}


def _plain_product(s):
    x = s["x"]
    dtype = x.dtype
    if "w" in s:
        w8 = _rounded(s["w"])
    else:
        w8 = _dequantize(s["codes"], s["scales"], x.shape[1])
    y = _rounded(x) @ w8.t()
    if "bias" in s:
        y = y + s["bias"].float()
    if s["case"]["relu"]:
        y = y.clamp_min(0)
    out = {"y": y.to(dtype)}
    if "dy" in s:
        dy = s["dy"]
        out["dx"] = (_rounded(dy) @ _rounded(s["w"].t()).t()).to(dtype)
        out["dw"] = (_rounded(dy.t()) @ _rounded(x.t()).t()).to(dtype)
        if "bias" in s:
            out["db"] = dy.double().sum(0).to(dtype)
    return out


def _noise(s, step):
    """32 bits for every element of the arena from its place in its tensor and the step: a multiplicative hash, finished by two
    rounds of xor-shift and multiply."""
    dev = s["p"].device
    padded = torch.tensor(s["padded"], device=dev)
    starts = torch.repeat_interleave(torch.tensor(s["starts"], device=dev), padded)
    i = torch.arange(s["p"].numel(), device=dev) - starts
    low = 0xFFFFFFFF
    h = (i * 0x9E3779B1 + (i >> 32) * 0xC2B2AE3D + step * 0x85EBCA77) & low
    h = h ^ (h >> 16)
    h = (h * 0x7FEB352D) & low
    h = h ^ (h >> 15)
    h = (h * 0x846CA68B) & low
    return h ^ (h >> 16)


def _stochastic(u, noise, bits, least):
    """u >= 0 to the neighbour below or above on a grid of `bits` mantissa bits (steps of 2^least below 2^(least + bits)): above with
    the probability of the remainder; noise: 16 bits."""
    _, ex = torch.frexp(u)
    step = _power((ex - 1 - bits).clamp_min(least))
    return torch.floor(u / step + noise / 65536.0) * step


def _plain_update(s):
    s["step"] += 1
    t = s["step"]
    bc1, bc2 = 1 - BETA1 ** t, 1 - BETA2 ** t
    g = s["g"].float()
    narrow = "master" in s
    p = torch.where(s["master"].to(s["p"].dtype) == s["p"], s["master"], s["p"].float()) if narrow else s["p"]
    if "scale" in s:
        sm, sv = s["scale"][:, :1], s["scale"][:, 1:]
        m = (s["m"].float().view(-1, BLOCK) * sm).view(-1)
        v = (s["v"].float().view(-1, BLOCK) * sv).view(-1)
    else:
        m, v = s["m"], s["v"]
    m = m + (1 - BETA1) * (g - m)
    v = v + (1 - BETA2) * (g * g - v)
    p = p - (LR * DECAY * p + LR / bc1 * m / (torch.sqrt(v) / math.sqrt(bc2) + EPS))
    if narrow:
        s["master"] = p
    s["p"] = p.to(s["p"].dtype)
    if "scale" in s:
        mb, vb = m.view(-1, BLOCK), v.view(-1, BLOCK)
        sm, sv = mb.abs().amax(1, keepdim=True) / 448, vb.amax(1, keepdim=True) / 57344
        h = _noise(s, t).view(-1, BLOCK)
        mu = _stochastic((mb.abs() / sm.clamp_min(1e-38)).clamp_max(448), (h & 0xFFFF).float(), 3, -9)
        vu = _stochastic((vb / sv.clamp_min(1e-38)).clamp_max(57344), (h >> 16).float(), 2, -16)
        vu = torch.where(vb > 0, vu.clamp_min(2.0 ** -16), vu)
        s["scale"] = torch.cat([sm, sv], 1)
        s["m"] = torch.copysign(mu, mb).to(torch.float8_e4m3fn).view(-1)
        s["v"] = vu.to(torch.float8_e5m2).view(-1)
    else:
        s["m"], s["v"] = m, v
    return {key: s[key] for key in ("p", "master", "m", "v", "scale") if key in s}


# ------------------------------------------------------------------------------------------------
# the framework's calls
# ------------------------------------------------------------------------------------------------
def _own_norm(s):
    from nerf_amd import ops
    if "dy" not in s:
        with torch.no_grad():
            return {"y": ops.layer_norm(s["x"], s["w"], s["b"])}
    x, w, b = (s[key].detach().requires_grad_(True) for key in ("x", "w", "b"))
    y = ops.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


def _own_product(s):
    from nerf_amd import ops
    bias, relu = s.get("bias"), s["case"]["relu"]
    if "dy" not in s:
        with torch.no_grad():
            return {"y": ops.linear_fp8(s["x"], ops.Fp8Rows(s["codes"], s["scales"], s["x"].shape[1]), bias, relu)}
    leaves = [t.detach().requires_grad_(True) for t in (s["x"], s["w"], bias) if t is not None]
    y = ops.linear_fp8(leaves[0], leaves[1], leaves[2] if bias is not None else None, relu)
    return dict(zip(("y", "dx", "dw", "db"), (y.detach(),) + torch.autograd.grad(y, leaves, s["dy"])))


def _own_update(s):
    from nerf_amd import optim
    if "optimizer" not in s:      # the object a training program keeps, resumed from the states at hand
        def cut(key, i, block=1):
            a = s["starts"][i] // block
            return s[key][a:a + -(-s["counts"][i] // block)]
        params = [torch.nn.Parameter(cut("p", i).view(shape)) for i, shape in enumerate(s["shapes"])]
        for i, p in enumerate(params):
            p.grad = cut("g", i).view(p.shape)
        opt = optim.AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, state_bits=s["case"]["bits"])
        for i, p in enumerate(params):
            opt.state[p] = {"step": torch.tensor(float(s["step"]), device=p.device), "exp_avg": cut("m", i).view(p.shape),
                            "exp_avg_sq": cut("v", i).view(p.shape)}
            if "scale" in s:
                opt.state[p]["scale"] = cut("scale", i, BLOCK)
            if "master" in s:
                opt.state[p]["master"] = cut("master", i).view(p.shape)
        s["optimizer"] = opt
    s["optimizer"].step()
    return {key: s[key] for key in ("p", "master", "m", "v", "scale") if key in s}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "product": _own_product, "update": _own_update}[op](state)
    return {"norm": _plain_norm, "product": _plain_product, "update": _plain_update}[op](state)


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["type"] == "float32" else 2
    if case["op"] == "norm":
        cells = case["n"] * case["c"]
        if case["train"]:         # x and dy read, y and dx written
            return {"bytes": size * (4 * cells + 4 * case["c"]), "flops": 22 * cells}
        return {"bytes": size * (2 * cells + 2 * case["c"]), "flops": 8 * cells}
    if case["op"] == "product":
        m, k, n = case["m"], case["k"], case["n"]
        if case["train"]:         # x, w, dy read; y, dx, dw written
            return {"bytes": size * 2 * (m * k + n * k + m * n), "flops": 6.0 * m * k * n}
        return {"bytes": size * (m * k + m * n) + n * k * (1 + 1 / BLOCK), "flops": 2.0 * m * k * n}
    count = sum(math.prod(s) for s in _shapes(case))
    per = 3 * size + (8 if size == 2 else 0) + (16 if case["bits"] == 32 else 4 + 16 / BLOCK)
    return {"bytes": per * count, "flops": 20 * count}


# ------------------------------------------------------------------------------------------------
# from the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def _two_to(e):
    """2^e in 64 bits, from its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _eight_bit(x):
    """What each value of x [r, k] stands for after quantising along k, in 64 bits."""
    x = x.double()
    r, k = x.shape
    blocks = torch.nn.functional.pad(x, (0, -k % BLOCK)).reshape(r, -1, BLOCK)
    top = blocks.abs().amax(2, keepdim=True)
    e = torch.frexp(top / 448)[1]                               # 2^(e-1) <= top / 448 < 2^e
    scale = torch.where(top <= 448 * _two_to(e - 1), _two_to(e - 1), _two_to(e))
    u = blocks / scale
    step = _two_to(torch.frexp(u.abs().clamp_min(2.0 ** -6))[1] - 4)
    return (torch.round(u / step) * step * scale).reshape(r, -1)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x, w, b = (s[key].double() for key in ("x", "w", "b"))
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        xh = (x - mean) / (var + 1e-5).sqrt()
        out = {"y": w * xh + b}
        if case["train"]:
            dy = s["dy"].double()
            c = case["c"]
            g = dy * w
            out["dx"] = (c * g - g.sum(1, keepdim=True) - xh * (g * xh).sum(1, keepdim=True)) / (c * (var + 1e-5).sqrt())
            out["dw"], out["db"] = torch.einsum("nc,nc->c", dy, xh), dy.sum(0)
        return out
    if case["op"] == "product":
        x = s["x"]
        if case["train"]:
            w = _eight_bit(s["w"])
        else:
            blocks = s["codes"].shape[1] // BLOCK
            w = s["codes"].double() * _two_to(s["scales"][:, :blocks].long() - 127).repeat_interleave(BLOCK, 1)
            w = w[:, : case["k"]]
        y = torch.mm(_eight_bit(x), w.t().contiguous())
        if case["bias"]:
            y += s["bias"].double()
        if case["relu"]:
            y = torch.relu(y)
        out = {"y": y}
        if case["train"]:
            dy = s["dy"]
            out["dx"] = torch.mm(_eight_bit(dy), _eight_bit(s["w"].t()).t().contiguous())
            out["dw"] = torch.mm(_eight_bit(dy.t()), _eight_bit(x.t()).t().contiguous())
            if case["bias"]:
                out["db"] = dy.double().sum(0)
        return out
    t = s["step"] + 1
    g = s["g"].double()
    p = (s["master"] if "master" in s else s["p"]).double()
    m, v = s["m"].double(), s["v"].double()
    if "scale" in s:
        wide = s["scale"].double().repeat_interleave(BLOCK, 0)
        m, v = m * wide[:, 0], v * wide[:, 1]
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g ** 2
    p = p * (1 - LR * DECAY) - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
    out = {"p": p, "m": m, "v": v}
    if "master" in s:
        out["master"] = p
    if "scale" in s:              # the rounded states have no value of their own: the noise decides
        out["m"] = out["v"] = None
        out["scale"] = torch.stack([m.abs().view(-1, BLOCK).amax(1) / 448, v.view(-1, BLOCK).amax(1) / 57344], 1)
    return out
