"""Cases for timing the loss end and the optimizer end of a training step.

``cross_entropy``: softmax cross entropy of a linear head over a large vocabulary, from hidden states and head weight, with the
gradients of both (or, for scoring, the losses alone).  ``adamw``: one AdamW step over a list of tensors, with the two running
averages in 32 bits or in blocks of 8-bit floats.

``run`` computes the plain form (elementary torch operations in 32 bits) while ``own`` is false and calls the framework otherwise.
``exact`` is written from the definitions in 64 bits."""
import math

import torch

own = False

Z_COEF = 1e-4
BETA1, BETA2, EPS, LR, DECAY = 0.9, 0.95, 1e-8, 3e-4, 0.1
STEP, SEED = 11, 20240611
BLOCK = 128
LARGEST_CE = 3 * 8192 * 4096 * 128256  # products of the largest listed training case
LARGEST_BYTES = 7e9  # of an optimizer step


def listed():
    ce = {"op": "cross_entropy", "z": False, "train": False}
    ad = {"op": "adamw", "layers": 1, "vocab": 0, "bits": 32, "master": True, "grad": "float32"}
    return [
        # the loss of a single token: one decoding step being scored, the latency of a call
        {**ce, "name": "score one token", "tokens": 1, "hidden": 2048, "vocab": 128256},
        # a padded batch of answers in an evaluation, odd vocabulary
        {**ce, "name": "score ragged", "tokens": 333, "hidden": 768, "vocab": 50257, "z": True},
        # scoring a long document batch
        {**ce, "name": "score long", "tokens": 16384, "hidden": 2048, "vocab": 128256},
        # a training step of a small model on a short batch
        {**ce, "name": "train small", "tokens": 256, "hidden": 1024, "vocab": 49152, "train": True},
        # odd numbers of tokens and words, with the z term
        {**ce, "name": "train odd z", "tokens": 2047, "hidden": 768, "vocab": 50257, "train": True, "z": True},
        # one vocabulary shard of two, large vocabulary beside a small hidden size
        {**ce, "name": "train wide", "tokens": 4096, "hidden": 1024, "vocab": 151936, "train": True},
        # the benchmark's own head on a full micro-batch
        {**ce, "name": "train large", "tokens": 8192, "hidden": 4096, "vocab": 128256, "train": True},
        # a handful of odd small tensors: norms and biases, launch bound
        {**ad, "name": "adamw 32 tiny", "hidden": 129, "inter": 517},
        # masters and bf16 copies of some layers of a 1B model
        {**ad, "name": "adamw 32 layers", "layers": 4, "hidden": 2048, "inter": 8192},
        # the same two with 8-bit states
        {**ad, "name": "adamw 8 tiny", "hidden": 129, "inter": 517, "bits": 8},
        # many layers of a small model trained without masters, bf16 gradients
        {**ad, "name": "adamw 8 bf16 many", "layers": 24, "hidden": 576, "inter": 1536, "vocab": 49152, "bits": 8, "master": False, "grad": "bfloat16"},
        # layers of the benchmark's own model, 8-bit states
        {**ad, "name": "adamw 8 large", "layers": 2, "hidden": 4096, "inter": 14336, "bits": 8},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        train = rng.random() < 0.6
        hidden = 64 * _log(rng, 1, 64)
        vocab = _log(rng, 200, 152000)
        most = LARGEST_CE // ((3 if train else 1) * hidden * vocab)
        tokens = _log(rng, 1, max(1, min(16384, most)))
        return {"op": "cross_entropy", "tokens": tokens, "hidden": hidden, "vocab": vocab, "train": train, "z": rng.random() < 0.3}
    bits, master = rng.choice((8, 32)), rng.random() < 0.6
    while True:
        case = {"op": "adamw", "layers": _log(rng, 1, 24), "hidden": _log(rng, 48, 4096), "inter": _log(rng, 64, 14336),
                "vocab": rng.choice((0, 0, _log(rng, 200, 50257))), "bits": bits, "master": master, "grad": "float32" if master else "bfloat16"}
        if work(case)["bytes"] <= LARGEST_BYTES:
            return case


def work(case):
    if case["op"] == "cross_entropy":
        t, h, v = case["tokens"], case["hidden"], case["vocab"]
        read = 2 * (t * h + v * h) + 8 * t
        if case["train"]:
            return {"bytes": read + 4 * t + 4 * t + 2 * (t * h + v * h), "flops": 6.0 * t * h * v}
        return {"bytes": read + 4 * t, "flops": 2.0 * t * h * v}
    n = sum(_sizes(case))
    param = 4 + 4 + 2 if case["master"] else 2 + 2
    grad = 4 if case["grad"] == "float32" else 2
    state = 16 if case["bits"] == 32 else 4 + 4 / BLOCK
    return {"bytes": n * (param + grad + state), "flops": 16.0 * n}


# ------------------------------------------------------------------------------------------------ inputs
def _sizes(case):
    """Elements of every tensor: per layer two norms, the attention and the gated MLP projections; then an embedding."""
    h, i = case["hidden"], case["inter"]
    kv = max(1, h // 4)
    sizes = [h, h * (h + 2 * kv), h * h, h, 2 * h * i, h * i] * case["layers"]
    return sizes + ([case["vocab"] * h] if case["vocab"] else [])


def _slots(case):
    """Where every tensor lies in the buffer of its kind: starts are multiples of BLOCK, as an allocator's are."""
    at, slots = 0, []
    for n in _sizes(case):
        slots.append((at, n))
        at += -(-n // BLOCK) * BLOCK
    return slots, at


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    if case["op"] == "cross_entropy":
        t, h, v = case["tokens"], case["hidden"], case["vocab"]
        x = (randn(t, h) * (0.7 + 0.6 * torch.rand(t, 1, generator=gen, device="cuda"))).to(torch.bfloat16)  # normalised hidden states
        w = torch.empty(v, h, dtype=torch.bfloat16, device="cuda")
        w.normal_(0.0, 1.5 / math.sqrt(h), generator=gen)
        y = torch.randint(0, v, (t,), generator=gen, device="cuda")
        mask = (torch.rand(t, generator=gen, device="cuda") < 0.95).float()  # the others are padding or prompt
        mask[0] = 1.0
        return {"case": case, "x": x, "w": w, "y": y, "g": mask / mask.sum()}
    slots, total = _slots(case)
    p = randn(total) * 0.02
    g = randn(total)
    g = (g * 1e-3 * torch.exp2(2.0 * randn(total // BLOCK).repeat_interleave(BLOCK))).to(getattr(torch, case["grad"]))
    g[torch.rand(total, generator=gen, device="cuda") < 0.01] = 0  # rows of the embedding that no token used
    m, v = g.float() * 0.3 + randn(total) * 2e-4, (randn(total) * 1e-3 + g.float() * 0.5).square()
    pad = torch.ones(total, dtype=torch.bool, device="cuda")
    for at, n in slots:
        pad[at : at + n] = False
    p[pad], g[pad], m[pad], v[pad] = 0, 0, 0, 0
    s = {"case": case, "scale": torch.full((1,), 0.83, device="cuda")}  # the clipping coefficient, a device scalar
    flat = {"grad": g}
    if case["master"]:
        flat["param"], flat["half"] = p, p.to(torch.bfloat16)
    else:
        flat["param"] = p.to(torch.bfloat16)
    if case["bits"] == 8:
        half = torch.full((total,), 0x8000, dtype=torch.int64, device="cuda")
        flat["m"], flat["m_exp"] = _encode(m, half, signed=True)
        flat["v"], flat["v_exp"] = _encode(v, half, signed=False)
    else:
        flat["m"], flat["v"] = m, v
    s["flat"] = flat
    s["list"] = {k: [f[at // BLOCK : (at + n + BLOCK - 1) // BLOCK] if k.endswith("_exp") else f[at : at + n] for at, n in slots] for k, f in flat.items()}
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if case["op"] == "cross_entropy":
        return _own_cross_entropy(state) if own else _plain_cross_entropy(state)
    if own:
        _own_adamw(state)
    else:
        for i in range(len(state["list"]["param"])):
            _plain_adamw(state, i)
    flat = state["flat"]
    out = {"param": flat["param"]}
    if case["master"]:
        out["half"] = flat["half"]
    if case["bits"] == 32:
        return {**out, "m": flat["m"], "v": flat["v"]}
    if own:
        from nanotron_b200 import ops

        # an 8-bit value has four significant bits and a power of two: bf16 holds it exactly
        m = ops.q8_decode(flat["m"], flat["m_exp"], signed=True, dtype=torch.bfloat16)
        v = ops.q8_decode(flat["v"], flat["v_exp"], signed=False, dtype=torch.bfloat16)
    else:
        m, v = _decode(flat["m"], flat["m_exp"], signed=True).to(torch.bfloat16), _decode(flat["v"], flat["v_exp"], signed=False).to(torch.bfloat16)
    return {**out, "m": m, "v": v}


def _own_cross_entropy(s):
    from nanotron_b200.parallel.tensor_parallel.functional import linear_cross_entropy, linear_cross_entropy_with_z_loss

    case, x, w = s["case"], s["x"], s["w"]
    if case["train"]:
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    if case["z"]:
        loss, z = linear_cross_entropy_with_z_loss(x, w, s["y"], z_loss_coef=Z_COEF)
    else:
        loss, z = linear_cross_entropy(x, w, s["y"]), None
    out = {"loss": loss.detach()}
    if z is not None:
        out["z"] = z.detach()
    if case["train"]:
        outputs = (loss,) if z is None else (loss, z)
        out["dx"], out["dw"] = torch.autograd.grad(outputs, (x, w), grad_outputs=(s["g"],) * len(outputs))
    return out


def _plain_cross_entropy(s):
    case, x, w, y = s["case"], s["x"].float(), s["w"].float(), s["y"]
    logits = x @ w.t()
    top = logits.max(dim=1, keepdim=True).values
    logz = top.squeeze(1) + torch.exp(logits - top).sum(dim=1).log()
    rows = torch.arange(y.numel(), device=y.device)
    out = {"loss": logz - logits[rows, y]}
    if case["z"]:
        out["z"] = Z_COEF * logz.square()
    if case["train"]:
        g = s["g"]
        coef = g + 2.0 * Z_COEF * logz * g if case["z"] else g
        d = torch.exp(logits - logz.unsqueeze(1)) * coef.unsqueeze(1)
        d[rows, y] -= g
        out["dx"], out["dw"] = (d @ w).to(torch.bfloat16), (d.t() @ x).to(torch.bfloat16)
    return out


def _own_adamw(s):
    from nanotron_b200 import ops

    t = s["list"]
    ops.adamw_multi_tensor(t["param"], t["grad"], t["m"], t["v"], halves=t.get("half"), exp_avg_exponents=t.get("m_exp"), exp_avg_sq_exponents=t.get("v_exp"),
                           lr=LR, beta1=BETA1, beta2=BETA2, eps=EPS, weight_decay=DECAY, step=STEP, grad_scale=s["scale"], seed=SEED)


def _plain_adamw(s, i):
    case, t = s["case"], {k: v[i] for k, v in s["list"].items()}
    eight = case["bits"] == 8
    m, v = (_decode(t["m"], t["m_exp"], signed=True), _decode(t["v"], t["v_exp"], signed=False)) if eight else (t["m"], t["v"])
    g = t["grad"].float() * s["scale"]
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    denom = v.sqrt() * (1.0 / math.sqrt(1 - BETA2**STEP)) + EPS
    p = t["param"].float() * (1 - LR * DECAY) - (LR / (1 - BETA1**STEP)) * (m / denom)
    t["param"].copy_(p)
    if case["master"]:
        t["half"].copy_(p)
    if eight:
        bits = _bits(m.numel(), i, m.device)
        for name, value, b in (("m", m, bits & 0xFFFF), ("v", v, bits >> 16)):
            codes, exponents = _encode(value, b, signed=name == "m")
            t[name].copy_(codes)
            t[name + "_exp"].copy_(exponents)
    else:
        t["m"].copy_(m)
        t["v"].copy_(v)


# ------------------------------------------------------------------------------------------------ 8-bit blocks, plainly
def _mix(x):
    """A 32-bit mixing function (two multiplications, three shifts) on int64 tensors or Python integers below 2^32."""
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _bits(n, tensor, device):
    """32 random bits for every element of the call's tensor number ``tensor`` (fewer than 2^32 elements)."""
    key = _mix((SEED + 0x9E3779B9 * (tensor + 1)) & 0xFFFFFFFF)
    return _mix(torch.arange(n, device=device) ^ key)


def _blocks(x):
    n = x.numel()
    return torch.nn.functional.pad(x, (0, -n % BLOCK)).view(-1, BLOCK)


def _encode(x, bits16, signed):
    """(codes, exponents): every block of 128 shares the fp32 exponent field E of its largest magnitude.  Code c > 0 (7 bits beside
    the sign, or 8 bits) counts eighths of binades from the window's lower end; the 20 cut mantissa bits round up with the
    probability that they stand for."""
    top = 127 if signed else 255
    raw = _blocks(x).contiguous().view(torch.int32).to(torch.int64)
    size = raw & 0x7FFFFFFF
    e = (size >> 23).amax(dim=1, keepdim=True)
    c = ((size + (_blocks(bits16) << 4) + 8) >> 20) - 8 * e + (top - 7)
    c = c.clamp(max=top)
    c = c.clamp(min=0 if signed else 1)  # a running mean of squares never becomes zero by rounding
    c = torch.where((size < 1 << 23) | (e == 255), torch.zeros_like(c), c)
    if signed:
        c = torch.where((c > 0) & (raw < 0), c + 128, c)
    return c.view(-1)[: x.numel()].to(torch.uint8), e.view(-1).to(torch.uint8)


def _decode(codes, exponents, signed):
    top = 127 if signed else 255
    c, e = _blocks(codes).to(torch.int64), exponents.to(torch.int64).unsqueeze(1)
    size = (c & top) + 8 * e - (top - 7)
    size = torch.where(((c & top) == 0) | (size < 8), torch.zeros_like(size), size)
    x = (size << 20).to(torch.int32).view(torch.float32)
    x = torch.where(c > top, -x, x)
    x = torch.where(e == 255, torch.full_like(x, math.nan), x)
    return x.view(-1)[: codes.numel()]


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_cross_entropy(s) if case["op"] == "cross_entropy" else _exact_adamw(s)


def _exact_cross_entropy(s):
    case, x, w, y, g = s["case"], s["x"].double(), s["w"], s["y"], s["g"].double()
    v, t = w.shape[0], x.shape[0]
    part = max(1, (1 << 28) // max(1, t))  # 2 GB of scores at a time
    logz, picked = torch.full((t,), -math.inf, dtype=torch.float64, device=x.device), torch.zeros(t, dtype=torch.float64, device=x.device)
    for a in range(0, v, part):
        scores = torch.einsum("th,vh->tv", x, w[a : a + part].double())
        logz = torch.logaddexp(logz, scores.logsumexp(dim=1))
        here = (y >= a) & (y < a + part)
        picked = torch.where(here, scores.gather(1, (y - a).clamp(0, scores.shape[1] - 1)[:, None])[:, 0], picked)
    out = {"loss": logz - picked}
    if case["z"]:
        out["z"] = Z_COEF * logz**2
    if case["train"]:
        out["dx"], out["dw"] = torch.zeros_like(x), torch.empty(w.shape, dtype=torch.float64, device=x.device)
        for a in range(0, v, part):
            piece = w[a : a + part].double()
            prob = torch.exp(torch.einsum("th,vh->tv", x, piece) - logz[:, None])
            grad = prob * (g * (1 + 2 * Z_COEF * logz) if case["z"] else g)[:, None]
            grad -= torch.nn.functional.one_hot((y - a).clamp(0, piece.shape[0] - 1), piece.shape[0]) * torch.where((y >= a) & (y < a + part), g, torch.zeros_like(g))[:, None]
            out["dx"] += torch.einsum("tv,vh->th", grad, piece)
            out["dw"][a : a + part] = torch.einsum("tv,th->vh", grad, x)
    return out


def _exact_adamw(s):
    case, flat = s["case"], {k: f.double() for k, f in s["flat"].items() if not k.endswith("_exp") and f.dtype != torch.uint8}
    eight = case["bits"] == 8
    if eight:
        for name in ("m", "v"):
            window = 15 if name == "m" else 31
            code, unit = s["flat"][name].double(), torch.exp2(s["flat"][name + "_exp"].double() - 127 - window).repeat_interleave(BLOCK)
            sign = torch.where(code > 127, -1.0, 1.0) if name == "m" else 1.0
            code = code % 128 if name == "m" else code
            flat[name] = torch.where(code > 0, sign * unit * torch.exp2((code / 8).floor()) * (1 + code % 8 / 8), 0.0)
    g = flat["grad"] * s["scale"].double()
    m, v = BETA1 * flat["m"] + (1 - BETA1) * g, BETA2 * flat["v"] + (1 - BETA2) * g**2
    p = flat["param"] - LR * DECAY * flat["param"] - LR * (m / (1 - BETA1**STEP)) / ((v / (1 - BETA2**STEP)) ** 0.5 + EPS)
    out = {"param": p}
    if case["master"]:
        out["half"] = p
    if eight:
        slots, total = _slots(case)
        bits = torch.zeros(total, dtype=torch.int64, device=p.device)
        for i, (at, n) in enumerate(slots):
            bits[at : at + n] = _bits(n, i, p.device)
        m, v = _exact_q8(m, bits & 0xFFFF, 15, False), _exact_q8(v, bits >> 16, 31, True)
    return {**out, "m": m, "v": v}


def _exact_q8(x, bits16, window, keep):
    """Every value of a block between two neighbours of the grid goes to the upper one when its share of the gap plus the random share
    reaches one."""
    size = x.abs().view(-1, BLOCK)
    top = torch.floor(torch.log2(size.amax(dim=1, keepdim=True).clamp(min=2.0**-126)))
    own_exp = torch.floor(torch.log2(size.clamp(min=2.0**-300)))
    gap = torch.exp2(own_exp) / 8
    share = (bits16.view(-1, BLOCK).double() * 16 + 8) / 2**20
    q = torch.floor(size / gap + share) * gap
    least = torch.exp2(top - window) * 1.125
    q = torch.minimum(q, torch.exp2(top) * 1.875)
    q = torch.where(q < least, torch.where(size > 0, least, 0.0) if keep else torch.zeros_like(q), q)
    return (q * x.view(-1, BLOCK).sign()).view(-1)
