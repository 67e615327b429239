"""AdamW over lists of tensors with 32- and 8-bit states: the 8-bit format, the PyTorch form and the kernel against the definition in 64
bits, the optimizer around them (state dicts, loading, masters), refusals, odd sizes, alignment, streams and captured graphs."""
import math

import pytest
import torch

from nanotron_b200 import ops
from nanotron_b200.ops import reference as ref
from nanotron_b200.optim.fused_adamw import FusedAdamW

gpu = pytest.mark.gpu
DEV = "cuda"
HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, step=3)


# ------------------------------------------------------------------------------------------------ the 8-bit format
def spread(n, seed=0, binades=3.0):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(n, generator=gen) * torch.exp2(binades * torch.randn(n, generator=gen))


@pytest.mark.parametrize("n", [1, 127, 128, 129, 1000])
@pytest.mark.parametrize("signed", [True, False])
def test_codes_round_trip_and_rounding_is_within_a_code(n, signed):
    x = spread(n) if signed else spread(n).square()
    c, e = ops.q8_encode(x, signed)
    assert c.dtype == e.dtype == torch.uint8 and c.shape == x.shape and e.shape == ((n + 127) // 128,)
    y = ops.q8_decode(c, e, signed)
    assert torch.equal(ops.q8_decode(c, e, signed, torch.bfloat16).float(), y)  # exact in bf16
    c2, e2 = ops.q8_encode(y, signed)
    assert torch.equal(c, c2) and torch.equal(e, e2)
    for b in range(0, n, 128):
        v, w = x[b : b + 128].double(), y[b : b + 128].double()
        top = 2.0 ** math.floor(math.log2(v.abs().max()))
        inside = v.abs() >= top * 2.0 ** (-15 if signed else -31) * 1.125
        # half an eighth of a binade; the largest code of the window can be short of its binade's end by one step
        assert ((w - v).abs()[inside] <= v.abs()[inside] / 16 * (1 + 2.0**-15) + (v.abs()[inside] >= top * 1.875) * top / 8).all()
        assert signed or (w > 0).all()  # a mean of squares never becomes zero by rounding


@pytest.mark.parametrize("signed", [True, False])
def test_special_blocks(signed):
    x = torch.zeros(128 * 5)
    x[128] = 2.0**-140                       # denormal only: zero
    x[2 * 128 : 2 * 128 + 3] = torch.tensor([1.0, 2.0**-40, 0.0])
    x[3 * 128] = math.inf
    x[4 * 128 + 5] = math.nan
    c, e = ops.q8_encode(x, signed)
    y = ops.q8_decode(c, e, signed)
    assert not y[:256].any() and y[256] == 1.0 and y[258] == 0.0
    assert (y[257] == 0.0) if signed else (y[257] == 2.0**-31 * 1.125)
    assert y[384:].isnan().all() and e[3] == e[4] == 255
    if signed:
        c, e = ops.q8_encode(-x[256:384], True)
        assert ops.q8_decode(c, e, True)[0] == -1.0


def test_stochastic_rounding_is_unbiased():
    """The mean over all 2^16 random shares is the value itself up to the share's resolution: 2^-16 of a code, a code being at most an
    eighth of the value."""
    for v in (1.0, 1.0625, 1.1, 1.3337, 1.9):
        r = torch.arange(1 << 16)
        x = torch.full((1 << 16,), v)
        x = torch.where(torch.arange(1 << 16) % 128 == 0, torch.tensor(4.0), x)  # the block's largest lies higher
        for signed in (True, False):
            y = ref.q8_decode(*ref.q8_encode(x, signed, r), signed)
            keep = r % 128 != 0
            assert abs(y[keep].double().mean().item() / float(x[1]) - 1) < 2.0**-3 * (2.0**-15 + 128 / 2**16), (v, signed)


def test_random_bits_are_uniform_enough():
    """Each of the 32 bits of 2^18 elements is one half of the time one: five standard deviations (2^-1 / 2^9 each)."""
    bits = ref.q8_random_bits(1 << 18, ref.q8_tensor_key(5, 2))
    for k in range(32):
        assert abs(((bits >> k) & 1).double().mean().item() - 0.5) < 5 * 0.5 / 2**9
    other = ref.q8_random_bits(1 << 18, ref.q8_tensor_key(6, 2))
    assert ((bits >> 16) == (other >> 16)).double().mean() < 2 * 2.0**-16 + 1e-3


# ------------------------------------------------------------------------------------------------ one step
def make(sizes, device, p_dtype, g_dtype, bits, half, seed=0, offset=0):
    """Lists of tensors for a step; ``offset``: every tensor starts that many elements into its storage."""
    gen = torch.Generator().manual_seed(seed)

    def place(t):
        if not offset:
            return t.to(device)
        out = torch.zeros(t.numel() + offset, dtype=t.dtype, device=device)
        out[offset:] = t.reshape(-1).to(device)
        return out[offset:].view(t.shape)

    out = {k: [] for k in ("p", "g", "m", "v", "me", "ve", "h")}
    for n in sizes:
        g = torch.randn(n, generator=gen) * 1e-2 * torch.exp2(2 * torch.randn(n, generator=gen))
        m, v = g * 0.3 + 1e-3 * torch.randn(n, generator=gen), (1e-2 * torch.randn(n, generator=gen)).square()
        out["p"].append(place(torch.randn(n, generator=gen).to(p_dtype)))
        out["g"].append(place(g.to(g_dtype)))
        for name, value, signed in (("m", m, True), ("v", v, False)):
            if bits == 8:
                c, e = ref.q8_encode(value, signed)
                out[name].append(place(c))
                out[name + "e"].append(e.to(device))
            else:
                out[name].append(place(value))
        out["h"].append(place(torch.zeros(n, dtype=torch.bfloat16)) if half else None)
    return out


def apply(t, bits, scale=None, seed=7, **over):
    kw = dict(HYPER, **over)
    ops.adamw_multi_tensor(t["p"], t["g"], t["m"], t["v"], halves=t["h"], exp_avg_exponents=t["me"] if bits == 8 else None, exp_avg_sq_exponents=t["ve"] if bits == 8 else None,
                           grad_scale=scale, seed=seed, **kw)


def expect(t, i, bits, scale, **over):
    """(p, m, v, bound of p, bound of m, bound of v) in 64 bits, m and v unrounded.

    Bounds: m is two rounded products (each with a rounded constant) and a sum, after the scaled gradient: 4 roundings of its larger
    part; v has two more on the squared part.  The step divides by a root: the error of m over the denominator, and a few units (2^-20)
    of approximate root and division; p adds its own roundings (2^-23) and, in bf16, half a step (2^-8)."""
    kw = dict(HYPER, **over)
    p, g = t["p"][i].double().cpu(), t["g"][i].double().cpu()
    m = (ref.q8_decode(t["m"][i], t["me"][i], True) if bits == 8 else t["m"][i]).double().cpu()
    v = (ref.q8_decode(t["v"][i], t["ve"][i], False) if bits == 8 else t["v"][i]).double().cpu()
    g = g * (float(scale) if scale is not None else 1.0)
    lr, b1, b2 = kw["lr"], kw["beta1"], kw["beta2"]
    big = b1 * m.abs() + (1 - b1) * g.abs()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    denom = (v / (1 - b2 ** kw["step"])).sqrt() + kw["eps"]
    size = lr / (1 - b1 ** kw["step"])
    q = p * (1 - lr * kw["weight_decay"]) - size * m / denom
    bp = 2.0**-22 * p.abs() + size * (2.0**-21 * big + 2.0**-20 * m.abs()) / denom + 1e-35
    if t["p"][i].dtype == torch.bfloat16:
        bp = bp + 2.0**-8 * q.abs()
    return q, m, v, bp, 2.0**-21 * big + 1e-37, 2.0**-21 * v + 1e-37


def close(got, want, bound, what):
    off = ((got.double().cpu() - want).abs() / bound).max().item() if got.numel() else 0.0
    assert off <= 1.0, f"{what}: {off:.3g} of the bound"


def check_step(sizes, device, p_dtype, g_dtype, bits, half, offset=0, scale=None, seed=7):
    t = make(sizes, device, p_dtype, g_dtype, bits, half, offset=offset)
    sc = None if scale is None else torch.tensor([scale], device=device)
    want = [expect(t, i, bits, sc) for i in range(len(sizes))]
    apply(t, bits, sc, seed)
    for i, (q, m, v, bp, bm, bv) in enumerate(want):
        close(t["p"][i], q, bp, f"p {i}")
        if half:
            assert torch.equal(t["h"][i].float(), t["p"][i].to(torch.bfloat16).float())
        if bits == 32:
            close(t["m"][i], m, bm, f"m {i}")
            close(t["v"][i], v, bv, f"v {i}")
        elif m.numel():
            r = ref.q8_random_bits(m.numel(), ref.q8_tensor_key(seed, i))
            for name, value, share, signed in (("m", m, r & 0xFFFF, True), ("v", v, r >> 16, False)):
                codes, exps = ref.q8_encode(value.float(), signed, share)
                # where fp32 rounding of the value changes the code it is the neighbour's: 2^-22 of the value against 2^-4
                differ = (codes != t[name][i].cpu()).double().mean().item()
                assert differ <= 1 / m.numel() + 1e-3, (name, i, differ)
                assert torch.equal(exps, t[name + "e"][i].cpu())


SIZES = [1, 3, 127, 128, 129, 0, 4096, 4097, 10007]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("p_dtype,g_dtype,half", [(torch.float32, torch.float32, True), (torch.bfloat16, torch.bfloat16, False), (torch.float32, torch.bfloat16, False)])
def test_pytorch_form_matches_the_definition(bits, p_dtype, g_dtype, half):
    check_step(SIZES, "cpu", p_dtype, g_dtype, bits, half, scale=0.7)


def test_matches_torch_adamw_over_steps():
    t = make([50, 7], "cpu", torch.float32, torch.float32, 32, False)
    for m, v in zip(t["m"], t["v"]):
        m.zero_(), v.zero_()
    theirs = [torch.nn.Parameter(p.clone()) for p in t["p"]]
    opt = torch.optim.AdamW([{"params": [theirs[0]], "lr": 1e-2, "weight_decay": 0.1}, {"params": [theirs[1]], "lr": 2e-2, "weight_decay": 0.0}], betas=(0.9, 0.95), eps=1e-8)
    for step in range(1, 4):
        for a, b in zip(theirs, t["g"]):
            a.grad = b * step
        opt.step()
        ops.adamw_multi_tensor(t["p"], [g * step for g in t["g"]], t["m"], t["v"], lr=[1e-2, 2e-2], weight_decay=[0.1, 0.0], beta1=0.9, beta2=0.95, eps=1e-8, step=step)
    for a, b in zip(theirs, t["p"]):
        torch.testing.assert_close(a.data, b, rtol=1e-5, atol=1e-6)


def test_refusals():
    ok = lambda: make([5, 200], "cpu", torch.float32, torch.float32, 8, True)  # noqa: E731

    def refused(change, bits=8, **kw):
        t = ok() if bits == 8 else make([5, 200], "cpu", torch.float32, torch.float32, 32, True)
        change(t)
        before = [p.clone() for p in t["p"]]
        with pytest.raises(ValueError):
            apply(t, bits, **kw)
        assert all(torch.equal(a, b) for a, b in zip(before, t["p"]))

    refused(lambda t: t["g"].pop())
    refused(lambda t: t["me"].__setitem__(1, t["me"][1][:1]))
    refused(lambda t: t["m"].__setitem__(0, t["m"][0].float()))
    refused(lambda t: t["g"].__setitem__(0, t["g"][0].half()))
    refused(lambda t: t["g"].__setitem__(0, t["g"][0][:4]))
    refused(lambda t: t["h"].__setitem__(0, t["h"][0].float()))
    refused(lambda t: t["p"].__setitem__(1, torch.zeros(10, 20).t()))
    refused(lambda t: t["v"].__setitem__(1, t["v"][1].to("meta")))
    refused(lambda t: [t[k].__setitem__(1, t[k][0]) for k in t])  # the same tensor twice
    refused(lambda t: None, bits=32, step=0)
    refused(lambda t: None, bits=32, beta1=1.0)
    refused(lambda t: None, bits=32, lr=[1e-2])
    refused(lambda t: None, scale=torch.ones(2))
    refused(lambda t: t["ve"].clear())
    t = ok()
    with pytest.raises(ValueError):
        ops.adamw_multi_tensor(t["p"], t["g"], t["m"], t["v"], exp_avg_exponents=t["me"], **HYPER)
    with pytest.raises(ValueError):
        ops.q8_decode(t["m"][1], t["me"][0], True)
    with pytest.raises(ValueError):
        ops.q8_decode(t["m"][1], t["me"][1], True, torch.float16)
    with pytest.raises(ValueError):
        ops.q8_encode(torch.zeros(3, dtype=torch.float64), True)
    with pytest.raises(ValueError):
        FusedAdamW([torch.nn.Parameter(torch.zeros(2))], state_bits=4)
    ops.adamw_multi_tensor([], [], [], [], **HYPER)


def test_values_that_are_not_finite_stay_in_their_block():
    t = make([300], "cpu", torch.float32, torch.float32, 8, False)
    t["g"][0][130] = math.inf
    apply(t, 8)
    m, v = ref.q8_decode(t["m"][0], t["me"][0], True), ref.q8_decode(t["v"][0], t["ve"][0], False)
    for x in (m, v):
        assert x[:128].isfinite().all() and x[256:].isfinite().all() and x[128:256].isnan().all()
    assert t["p"][0].isfinite().sum() == 299


# ------------------------------------------------------------------------------------------------ the optimizer
def model_params(device="cpu", dtype=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(*s, generator=gen).to(device, dtype)) for s in ((30, 17), (129,), (4, 64))]


def steps(opt, params, n, seed=1, first=0):
    for k in range(first, first + n):
        gen = torch.Generator().manual_seed(seed + 100 * k)
        for p in params:
            p.grad = (torch.randn(p.shape, generator=gen) * 0.1).to(p.device, p.dtype)
        opt.step()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_8_bit_optimizer_saves_and_resumes_bit_for_bit(device):
    a, b = model_params(device), model_params(device)
    opt_a, opt_b = (FusedAdamW([{"params": x[:2], "weight_decay": 0.1}, {"params": x[2:], "weight_decay": 0.0}], lr=1e-2, state_bits=8) for x in (a, b))
    steps(opt_a, a, 3)
    assert all(s["exp_avg"].dtype == torch.uint8 for s in opt_a.state.values())
    saved = {k: v for k, v in opt_a.state_dict().items()}
    st = saved["state"][0]
    assert set(st) == {"step", "exp_avg", "exp_avg_sq"} and st["exp_avg"].dtype == torch.float32 and st["exp_avg"].shape == a[0].shape
    for x, y in zip(a, b):
        y.data.copy_(x.data)
    opt_b.load_state_dict(torch.utils._pytree.tree_map(lambda v: v.cpu().clone() if torch.is_tensor(v) else v, saved))
    steps(opt_a, a, 2, first=3), steps(opt_b, b, 2, first=3)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
        for key in ("exp_avg", "exp_avg_exponents", "exp_avg_sq", "exp_avg_sq_exponents"):
            assert torch.equal(opt_a.state[x][key], opt_b.state[y][key])


def test_8_bit_optimizer_reads_a_32_bit_state_and_back():
    a, b = model_params(), model_params()
    full, small = FusedAdamW(a, lr=1e-2), FusedAdamW(b, lr=1e-2, state_bits=8)
    steps(full, a, 2), steps(small, b, 2)
    small.load_state_dict(full.state_dict())
    steps(small, b, 1, first=2)
    for x, y in zip(a, b):
        m = full.state[x]["exp_avg"]
        got = ref.q8_decode(small.state[y]["exp_avg"], small.state[y]["exp_avg_exponents"], True)
        assert got.shape == m.shape and small.state[y]["step"] == 3
    full.load_state_dict(small.state_dict())
    assert torch.equal(full.state[a[0]]["exp_avg"], ref.q8_decode(small.state[b[0]]["exp_avg"], small.state[b[0]]["exp_avg_exponents"], True))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_8_bit_first_step_is_the_32_bit_one(device):
    """From a fresh state the step uses the unrounded averages: nothing of the 8-bit form shows yet."""
    a, b = model_params(device), model_params(device)
    steps(FusedAdamW(a, lr=1e-2), a, 1), steps(FusedAdamW(b, lr=1e-2, state_bits=8), b, 1)
    for x, y in zip(a, b):
        torch.testing.assert_close(x, y, rtol=2.0**-20, atol=1e-2 * 2.0**-19)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("devices", [("cpu", "cpu"), pytest.param((DEV, "cpu"), marks=gpu)])
def test_gradient_scale_of_any_kind_and_parameters_on_two_devices(bits, devices):
    """The scale may be a number, or a scalar of another type or device than the parameters; 0.5 is exact in all of them."""

    def stepped(scale, factor):
        params = [torch.nn.Parameter((torch.arange(300.0) / 300).to(d)) for d in devices]
        opt = FusedAdamW(params, lr=1e-2, state_bits=bits)
        opt.grad_scale = scale
        for p in params:
            p.grad = torch.linspace(-1, 1, 300).to(p.device) * factor
        opt.step()
        return [p.detach().cpu() for p in params]

    want = stepped(None, 0.5)
    for scale in (0.5, torch.tensor(0.5), torch.tensor([0.5], dtype=torch.float64), torch.tensor(0.5, device=devices[0])):
        for a, b in zip(stepped(scale, 1.0), want):
            assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ GPU
@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("p_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("g_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("half,offset", [(True, 0), (False, 0), (True, 1), (True, 4)])
def test_kernel_matches_the_definition(bits, p_dtype, g_dtype, half, offset):
    check_step(SIZES, DEV, p_dtype, g_dtype, bits, half, offset=offset, scale=0.7)


@gpu
@pytest.mark.parametrize("signed", [True, False])
@pytest.mark.parametrize("n", [1, 127, 128, 129, 70001])
def test_kernel_codes_equal_the_pytorch_ones(signed, n):
    x = spread(n, seed=4, binades=6.0) if signed else spread(n, seed=4, binades=6.0).square()
    x[n // 2] = 0.0
    c, e = ref.q8_encode(x, signed)
    for off in (0, 1):
        y = torch.zeros(n + off, device=DEV)
        y[off:] = x.to(DEV)
        cg, eg = ops.q8_encode(y[off:], signed)
        assert torch.equal(cg.cpu(), c) and torch.equal(eg.cpu(), e)
        for dtype in (torch.float32, torch.bfloat16):
            assert torch.equal(ops.q8_decode(cg, eg, signed, dtype).cpu(), ref.q8_decode(c, e, signed, dtype))


@gpu
@pytest.mark.parametrize("g_dtype", [torch.float32, torch.bfloat16])
def test_8_bit_states_equal_the_pytorch_form_over_steps(g_dtype):
    """m and v take separately rounded operations: the codes are the same bytes wherever the formula is evaluated."""
    a = make([5, 128, 70001], DEV, torch.float32, g_dtype, 8, False)
    b = {k: [x.cpu() if x is not None else None for x in v] for k, v in a.items()}
    for step in range(1, 6):
        for t in (a, b):
            apply(t, 8, torch.tensor(0.83, device=t["p"][0].device), seed=step, step=step)
    for k in ("m", "v", "me", "ve"):
        for x, y in zip(a[k], b[k]):
            assert torch.equal(x.cpu(), y), k


@gpu
def test_8_bit_states_equal_the_pytorch_form_on_many_elements():
    """A last bit of m or v changes a code with a chance of about 2^-20: 2^26 elements would show it if a share of the sums were rounded
    otherwise (by a fused multiply-add, say)."""
    n = 1 << 26
    gen = torch.Generator(device=DEV).manual_seed(5)
    g = torch.randn(n, generator=gen, device=DEV) * 1e-2
    m, v = g * 0.3 + 1e-3 * torch.randn(n, generator=gen, device=DEV), (1e-2 * torch.randn(n, generator=gen, device=DEV)).square()
    a = {"p": [torch.zeros(n, device=DEV)], "g": [g], "h": None}
    (c, e), (k, f) = ops.q8_encode(m, True), ops.q8_encode(v, False)
    a["m"], a["me"], a["v"], a["ve"] = [c], [e], [k], [f]
    b = {key: [t.clone() for t in value] if value else None for key, value in a.items()}
    scale = torch.tensor(0.83, device=DEV)
    apply(a, 8, scale)
    with ops.mode("torch"):
        apply(b, 8, scale)
    for key in ("m", "v", "me", "ve"):
        assert torch.equal(a[key][0], b[key][0]), key


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [24, 25, 384, 385, 800])
def test_many_tensors(bits, count):
    check_step([1 + (37 * i) % 300 for i in range(count)], DEV, torch.float32, torch.float32, bits, False)


@gpu
def test_32_bit_step_agrees_with_the_flat_kernel():
    """The flat kernel takes 1 - b from the fp32 b: off by 2^-25 / (1 - b), 2^-21.7 of m's and 2^-20.7 of v's new part."""
    from nanotron_b200.ops import native

    t = make([128 * 40, 128 * 9], DEV, torch.float32, torch.float32, 32, True)
    flat = {k: torch.cat([x.clone() for x in t[k]]) for k in ("p", "g", "m", "v", "h")}
    scale = torch.tensor([0.6], device=DEV)
    ends = torch.tensor([128 * 40, 128 * 49], dtype=torch.int64, device=DEV)
    native.adamw_flat(flat["p"], flat["g"], flat["m"], flat["v"], flat["h"], ends, torch.tensor([1e-2, 3e-3], device=DEV), torch.tensor([0.1, 0.0], device=DEV), 0.9, 0.95, 1e-8, 3, scale)
    apply(t, 32, scale, lr=[1e-2, 3e-3], weight_decay=[0.1, 0.0])
    for k, rtol, atol in (("m", 2.0**-20, 2.0**-24), ("v", 2.0**-19, 1e-30), ("p", 2.0**-21, 1e-2 * 2.0**-18), ("h", 2.0**-7, 1e-30)):
        torch.testing.assert_close(torch.cat(t[k]), flat[k], rtol=rtol, atol=atol)


@gpu
def test_special_gradients_on_the_gpu():
    a = make([300, 4096], DEV, torch.float32, torch.float32, 8, False)
    a["g"][0][130], a["g"][0][5], a["g"][1][:] = math.nan, 0.0, 0.0
    b = {k: [x.cpu() if x is not None else None for x in v] for k, v in a.items()}
    apply(a, 8), apply(b, 8)
    for k in ("m", "v", "me", "ve"):
        for x, y in zip(a[k], b[k]):
            assert torch.equal(x.cpu(), y), k
    assert a["p"][0].isfinite().sum() == 299


@gpu
def test_strided_gradients_and_mixed_types_in_one_call():
    t = make([600, 600, 128], DEV, torch.float32, torch.float32, 8, False)
    want = {k: [x.clone() if x is not None else None for x in v] for k, v in t.items()}
    apply(want, 8)
    t["g"][0] = t["g"][0].view(20, 30).t().contiguous().t()  # the same numbers through other strides
    t["p"][0], t["m"][0], t["v"][0] = (t[k][0].view(20, 30) for k in ("p", "m", "v"))
    apply(t, 8)
    assert torch.equal(t["p"][0].view(-1), want["p"][0]) and torch.equal(t["m"][0].view(-1), want["m"][0])
    mixed = make([600, 600, 128], DEV, torch.float32, torch.float32, 8, False)
    mixed["g"][1], mixed["p"][2] = mixed["g"][1].to(torch.bfloat16), mixed["p"][2].to(torch.bfloat16)
    before = [expect(mixed, i, 8, None) for i in range(3)]
    apply(mixed, 8)
    for i, (q, _, _, bp, _, _) in enumerate(before):
        close(mixed["p"][i], q, bp, f"p {i}")


@gpu
def test_captured_steps_and_other_streams():
    t = make([1000, 77], DEV, torch.float32, torch.float32, 8, True)
    u = {k: [x.clone() if x is not None else None for x in v] for k, v in t.items()}
    w = {k: [x.clone() if x is not None else None for x in v] for k, v in t.items()}
    scale = torch.tensor([0.5], device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        apply(t, 8, scale)
    junk = [torch.zeros(5000, device=DEV) for _ in range(8)]  # the table of a captured launch is the graph's own
    scale.fill_(0.25)
    graph.replay()
    apply(u, 8, scale)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        apply(w, 8, scale)
    torch.cuda.synchronize()
    del junk
    for k in ("p", "h", "m", "v", "me", "ve"):
        for x, y, z in zip(t[k], u[k], w[k]):
            assert torch.equal(x, y) and torch.equal(x, z), k


@gpu
def test_a_tensor_past_32_bits_of_elements():
    n = (1 << 32) + 200
    p, g = torch.zeros(n, dtype=torch.bfloat16, device=DEV), torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    m, v = torch.zeros(n, dtype=torch.uint8, device=DEV), torch.zeros(n, dtype=torch.uint8, device=DEV)
    me, ve = (torch.zeros((n + 127) // 128, dtype=torch.uint8, device=DEV) for _ in range(2))
    gen = torch.Generator().manual_seed(3)
    tail = (1 << 32) - 128
    values = torch.randn(n - tail, generator=gen).to(torch.bfloat16)
    g[tail:] = values.to(DEV)
    ops.adamw_multi_tensor([p], [g], [m], [v], exp_avg_exponents=[me], exp_avg_sq_exponents=[ve], seed=9, **dict(HYPER, step=1))
    index = torch.arange(tail, n)
    key = ref.q8_tensor_key(9, 0)
    bits = ref.mix32((index & 0xFFFFFFFF) ^ ((key + (index >> 32) * 0x9E3779B9) & 0xFFFFFFFF))
    x = values.float()
    for codes, exps, value, share, signed in ((m, me, x * (1 - 0.9), bits & 0xFFFF, True), (v, ve, (x * x) * (1 - 0.95), bits >> 16, False)):
        c, e = ref.q8_encode(value, signed, share)
        assert torch.equal(codes[tail:].cpu(), c) and torch.equal(exps[tail // 128 :].cpu(), e)
        assert not codes[: 1 << 20].any() and not exps[: tail // 128].any()
    assert (p[tail:].float().sign().cpu() == -x.sign()).all() and not p[: 1 << 20].any()


@gpu
def test_scattered_masters_take_one_launch():
    params = model_params(DEV)
    refs = [torch.nn.Parameter(p.detach().clone()) for p in params]
    half = [torch.zeros(p.numel(), dtype=torch.bfloat16, device=DEV) for p in params]
    opt, theirs = FusedAdamW(params, lr=1e-2, weight_decay=0.1), torch.optim.AdamW(refs, lr=1e-2, weight_decay=0.1)
    for p, h in zip(params, half):
        opt.set_half_target(p, h)
    steps(opt, params, 1), steps(theirs, refs, 1)
    n0 = ops.native_launches()
    steps(opt, params, 2, first=1), steps(theirs, refs, 2, first=1)
    assert ops.native_launches() - n0 == 2 and opt._flat is None
    for p, r, h in zip(params, refs, half):
        torch.testing.assert_close(p, r, rtol=1e-5, atol=1e-6)
        assert torch.equal(h, p.detach().view(-1).to(torch.bfloat16))
