"""The AdamW step over many tensors (`adamw_step_`, `AdamW`) against its definition on the host: in 64 bits for fp32 moments and
all parameters, bit for bit for 8-bit moments (whose fp32 arithmetic is a fixed sequence of rounded products and sums).

Tolerances.  fp32 moments: three roundings of 2^-24 and fp32 betas, 5 * 2^-24 of the summands' sizes, times the steps made.  A
parameter: two roundings of 2^-24 of itself, an update whose root, reciprocal, products and scalars are off by a few units of
2^-23 (1e-6 in all, plus half of what v is off by and what m is), and half a step of its type; in 16 bits a parameter that lies
between two values may go either way, so one whole step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = [(1,), (3,), (255,), (16, 16), (257,), (7, 33), (8192,), (8193,), (0,), (100, 1003), (65537,)]
B1, B2, EPS, WD, LR = 0.9, 0.999, 1e-8, 0.1, 1e-2


def make(sizes, dtype, seed, offset=0):
    """Tensors on the GPU, `offset` entries into their storage."""
    g = torch.Generator().manual_seed(seed)

    def put(x, t):
        store = torch.empty(x.numel() + offset, dtype=t, device=DEV)
        out = store[offset:].view(x.shape)
        out.copy_(x)
        return out

    p = [put(torch.randn(s, generator=g), dtype) for s in sizes]
    grads = [put(torch.randn(s, generator=g) * 10.0 ** float(torch.randint(-4, 1, (1,), generator=g)), dtype) for s in sizes]
    return p, grads, put


def zeros32(sizes, put):
    return [put(torch.zeros(s), torch.float32) for s in sizes], [put(torch.zeros(s), torch.float32) for s in sizes]


def step_counters(n, at=0.0):
    return [torch.full((), at, device=DEV) for _ in range(n)]


def norm64(grads):
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def definition(p, g, m, v, t, clip=1.0, lr=LR, wd=WD, b1=B1, b2=B2, eps=EPS):
    g = g.double().cpu() * clip
    m = b1 * m.double().cpu() + (1 - b1) * g
    v = b2 * v.double().cpu() + (1 - b2) * g * g
    update = (m / (1 - b1**t)) / ((v / (1 - b2**t)).sqrt() + eps)
    return p.double().cpu() * (1 - lr * wd) - lr * update, m, v, update


def check_param(got, p, want, update, dtype, lr=LR):
    bound = 2.0**-23 * want.abs() + 2e-6 * lr * update.abs() + torch.finfo(dtype).eps * want.abs() / (2 if dtype == torch.float32 else 1) + 1e-12
    if dtype == torch.float16:
        bound = bound + 2.0**-24  # (subnormal numbers)
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), (off - bound).max()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_fp32_moments(dtype, offset):
    import trl_amd

    t = DTYPES[dtype]
    p, grads, put = make(SIZES, t, 3, offset)
    m, v = zeros32(SIZES, put)
    steps = step_counters(len(SIZES))
    for i in range(1, 4):
        before = [x.clone() for x in p], [x.clone() for x in m], [x.clone() for x in v]
        assert trl_amd.adamw_step_(p, grads, m, v, steps, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD) is None
        for k in range(len(SIZES)):
            want_p, want_m, want_v, update = definition(before[0][k], grads[k], before[1][k], before[2][k], i)
            g = grads[k].double().cpu().abs()
            assert bool(((m[k].double().cpu() - want_m).abs() <= 5 * 2.0**-24 * (B1 * before[1][k].double().cpu().abs() + (1 - B1) * g) + 1e-44).all())
            assert bool(((v[k].double().cpu() - want_v).abs() <= 5 * 2.0**-24 * (want_v + (1 - B2) * g * g) + 1e-44).all())
            check_param(p[k], before[0][k], want_p, update, t)
        assert all(float(s) == i for s in steps)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_clipping_and_the_norm(dtype):
    import trl_amd

    t = DTYPES[dtype]
    for max_norm, expect_clip in ((0.5, True), (1e6, False), (0, False)):
        p, grads, put = make(SIZES, t, 5)
        m, v = zeros32(SIZES, put)
        before, kept = [x.clone() for x in p], [x.clone() for x in grads]
        norm = norm64(grads)
        got = trl_amd.adamw_step_(p, grads, m, v, step_counters(len(SIZES)), lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD,
                                  max_grad_norm=max_norm)
        assert got.shape == () and abs(float(got) - norm) <= 2.0**-24 * norm + 1e-12
        clip = max_norm / (norm + 1e-6) if expect_clip else 1.0
        assert (clip < 1) == expect_clip
        for k in range(len(SIZES)):
            assert torch.equal(grads[k], kept[k])
            want_p, want_m, want_v, update = definition(before[k], grads[k], torch.zeros(SIZES[k]), torch.zeros(SIZES[k]), 1, clip)
            torch.testing.assert_close(m[k].double().cpu(), want_m, rtol=6 * 2.0**-24, atol=1e-44)
            torch.testing.assert_close(v[k].double().cpu(), want_v, rtol=8 * 2.0**-24, atol=1e-44)
            check_param(p[k], before[k], want_p, update, t)


# ---- 8-bit moments ----------------------------------------------------------------------------------------------------
def mix(x):
    x = ((x ^ (x >> 16)) * 0x55CE65AD) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0xCDBE2AF7) & 0xFFFFFFFF
    return x ^ (x >> 16)


def random_bits(n, step, index, seed):
    salt = mix(mix(torch.tensor(int(step) ^ seed)) + 0x9E3779B9 * (index + 1) & 0xFFFFFFFF)
    return mix(salt + torch.arange(n) * 0x9E3779B1 & 0xFFFFFFFF)


def code_values(signed):
    """The 256 codes' values in units of the scale."""
    c = torch.arange(256)
    mantissa = 3 if signed else 4
    e, f = (c & (127 if signed else 255)) >> mantissa, c & (2**mantissa - 1)
    value = torch.where(e == 0, f * 2.0 ** (-6 - mantissa), (1 + f / 2.0**mantissa) * 2.0 ** (e - 7).float())
    return torch.where(c > 127, -value, value) if signed else value


def decode(codes, scales, signed):
    n = codes.numel()
    return code_values(signed)[codes.flatten().view(torch.uint8).long()] * scales.repeat_interleave(256)[:n]


def encode(x, signed, r16):
    """Codes by looking both neighbours up: up with the probability that keeps the mean, cut to 16 bits."""
    n = x.numel()
    blocks = torch.nn.functional.pad(x, (0, -n % 256)).view(-1, 256).abs().amax(1)
    scales = torch.where(blocks > 0, 2.0 ** torch.ceil(torch.log2(blocks.double() / 448)), 1.0).float()
    y = (x.abs().double() / scales.double().repeat_interleave(256)[:n])
    values = code_values(signed)[: 127 if signed else 253].double()
    low = torch.searchsorted(values, y, right=True) - 1
    high = (low + 1).clamp(max=len(values) - 1)
    step = values[high] - values[low]
    part = torch.where(step > 0, (y - values[low]) / torch.where(step > 0, step, 1.0), 0.0)
    # (the part between two codes, cut to 2^-20 of a step for normal codes and 2^-16 for small ones, plus the random bits)
    digits = 20 if signed else 19
    cut = torch.where(y < 2.0**-6, torch.floor(part * 2**16) * 2**-16, torch.floor(part * 2**digits) * 2**-digits)
    code = torch.where(cut + r16.double() * 2.0**-16 >= 1, high, low)
    if signed:
        return (code + 128 * (x < 0)).to(torch.uint8), scales
    return torch.where(y > 0, code.clamp(min=1), code).to(torch.uint8), scales


def eight_bit_state(sizes):
    n = [math.prod(s) for s in sizes]
    codes = [torch.zeros(s, dtype=torch.uint8, device=DEV) for s in sizes]
    return ([c.clone().view(torch.float8_e4m3fn) for c in codes], codes, [torch.ones(-(-k // 256), device=DEV) for k in n],
            [torch.ones(-(-k // 256), device=DEV) for k in n])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("offset", [0, 1])
def test_8bit_moments(dtype, offset):
    """Every code, scale and parameter of three steps, with and without clipping, from the state before the step."""
    import trl_amd

    t = DTYPES[dtype]
    p, grads, put = make(SIZES, t, 7, offset)
    grads[3][:] = 0.0  # (a block of zeros)
    grads[9][3] *= 1e-6 if dtype != "fp16" else 1e-2
    m, v, ms, vs = eight_bit_state(SIZES)
    if offset:
        m = [put(x.view(torch.uint8).float(), torch.uint8).view(torch.float8_e4m3fn) for x in m]
        v = [put(x.float(), torch.uint8) for x in v]
    steps, seed = step_counters(len(SIZES), 4.0), 77
    one = torch.ones((), dtype=torch.float32)
    for i, max_norm in enumerate((None, 0.7, 0.7)):
        before = [[x.cpu().clone() for x in xs] for xs in (p, m, v, ms, vs)]
        norm = trl_amd.adamw_step_(p, grads, m, v, steps, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, max_grad_norm=max_norm,
                                   exp_avg_scales=ms, exp_avg_sq_scales=vs, seed=seed)
        clip64 = 1.0 if max_norm is None else min(1.0, max_norm / (norm64(grads) + 1e-6))
        clip = one * clip64
        assert norm is None or abs(float(norm) - norm64(grads)) <= 2.0**-24 * norm64(grads)
        for k, s in enumerate(SIZES):
            if not math.prod(s):
                continue
            g = grads[k].cpu().float().flatten() * clip
            om, ov = decode(before[1][k], before[3][k], True), decode(before[2][k], before[4][k], False)
            nm = om * B1 + g * (1 - B1)
            nv = ov * B2 + g * g * (1 - B2)
            bits = random_bits(g.numel(), 5 + i, k, seed)
            for got, scales, x, signed, r in ((m[k], ms[k], nm, True, bits & 0xFFFF), (v[k], vs[k], nv, False, bits >> 16)):
                codes, want_scales = encode(x, signed, r)
                assert torch.equal(scales.cpu(), want_scales), (k, signed)
                assert torch.equal(got.cpu().view(torch.uint8).flatten(), codes), (k, signed)
                values = trl_amd.adamw_state_values(got, scales)
                assert torch.equal(values.cpu().float().flatten(), decode(codes, want_scales, signed)) and values.shape == got.shape
            want_p, _, _, update = definition(before[0][k].flatten(), grads[k].flatten(), om, ov, 5 + i, clip64)
            check_param(p[k].flatten(), before[0][k].flatten(), want_p, update, t)


def test_rounding_keeps_the_mean():
    """One value in every entry: the mean of its codes' values over many entries.  A rounding is off by at most a step, so the mean
    of n by 6 / sqrt(n) of one, and by 2^-16 of one because the random numbers have 16 bits."""
    import trl_amd

    n = 1 << 20
    for x in (1.03, 3.3e-2, 0.51):
        p, g = [torch.zeros(n, device=DEV)], [torch.full((n,), x, device=DEV)]
        g[0][::256] = 2.0  # the block's largest
        m, v, ms, vs = eight_bit_state([(n,)])
        trl_amd.adamw_step_(p, g, m, v, step_counters(1), betas=(B1, B2), exp_avg_scales=ms, exp_avg_sq_scales=vs, seed=5)
        rest = torch.ones(n, dtype=torch.bool, device=DEV)
        rest[::256] = False
        for values, want, step in ((trl_amd.adamw_state_values(m[0], ms[0]), 0.1 * x, 2.0**-3), (trl_amd.adamw_state_values(v[0], vs[0]), 1e-3 * x * x, 2.0**-4)):
            mean = float(values[rest].double().mean())
            assert len(values[rest].unique()) == 2
            assert abs(mean / want - 1) < step * (6 / math.sqrt(n) + 2.0**-16) + 2.0**-22


def test_8bit_second_moment_does_not_stand_still():
    """300 steps with gradients of one size: v grows as 1 - b2^t although a step moves it by less than a code.  v is a sum of its
    rounding errors, independent with mean 0 and at most half a step (2^-5 of v) each: standard deviation under sqrt(300) / 32 = 0.54
    of v, of a mean over 2^16 entries 0.0022."""
    import trl_amd

    n = 1 << 16
    p, g = [torch.zeros(n, device=DEV)], [torch.ones(n, device=DEV)]
    m, v, ms, vs = eight_bit_state([(n,)])
    steps = step_counters(1)
    for _ in range(300):
        trl_amd.adamw_step_(p, g, m, v, steps, lr=0.0, betas=(B1, B2), exp_avg_scales=ms, exp_avg_sq_scales=vs)
    mean = float(trl_amd.adamw_state_values(v[0], vs[0]).double().mean())
    assert abs(mean / (1 - B2**300) - 1) < 6 * 0.0022


def test_numbers_that_are_not_finite():
    import trl_amd

    for bad in (math.nan, math.inf):
        sizes = [(1000,), (500,)]
        p, g, put = make(sizes, torch.float32, 9)
        g[0][300] = bad
        m, v = zeros32(sizes, put)
        trl_amd.adamw_step_(p, g, m, v, step_counters(2))
        hit = torch.zeros(1000, dtype=torch.bool)
        hit[300] = True
        assert torch.equal(p[0].isnan().cpu(), hit) and not bool(p[1].isnan().any())
        assert torch.equal(m[0].isfinite().cpu(), ~hit) and torch.equal(v[0].isfinite().cpu(), ~hit)
        # 8 bits: the block
        p, g, put = make(sizes, torch.float32, 9)
        g[0][300] = bad
        m, v, ms, vs = eight_bit_state(sizes)
        trl_amd.adamw_step_(p, g, m, v, step_counters(2), exp_avg_scales=ms, exp_avg_sq_scales=vs)
        assert torch.equal(p[0].isnan().cpu(), hit)
        for c, s in ((m, ms), (v, vs)):
            values = trl_amd.adamw_state_values(c[0], s[0])
            assert bool(values[256:512].isnan().all()) and bool(values[:256].isfinite().all()) and bool(values[512:].isfinite().all())
        # clipping: a norm that is none reaches everything
        p, g, put = make(sizes, torch.float32, 9)
        g[0][300] = math.nan
        m, v = zeros32(sizes, put)
        norm = trl_amd.adamw_step_(p, g, m, v, step_counters(2), max_grad_norm=1.0)
        assert math.isnan(float(norm)) and bool(p[1].isnan().all())


def test_many_tensors_and_types_in_one_call():
    """More tensors than a launch takes, of three types, small and large: against torch's optimiser in 64 bits."""
    import trl_amd

    g = torch.Generator().manual_seed(11)
    p, grads, put = [], [], None
    for i in range(700):
        t = (torch.float32, torch.bfloat16, torch.float16)[i % 3]
        n = int(torch.randint(1, 3000, (1,), generator=g)) if i % 50 else 40000
        a, b, put = make([(n,)], t, 1000 + i)
        p += a
        grads += b
    sizes = [tuple(x.shape) for x in p]
    m, v = zeros32(sizes, put)
    before = [x.clone() for x in p]
    steps = step_counters(len(p))
    norm = trl_amd.adamw_step_(p, grads, m, v, steps, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, max_grad_norm=1.0)
    clip = min(1.0, 1.0 / (norm64(grads) + 1e-6))
    assert abs(float(norm) / norm64(grads) - 1) < 2.0**-23
    for k in range(len(p)):
        want_p, want_m, _, update = definition(before[k], grads[k], torch.zeros(sizes[k]), torch.zeros(sizes[k]), 1, clip)
        check_param(p[k], before[k], want_p, update, p[k].dtype)
        torch.testing.assert_close(m[k].double().cpu(), want_m, rtol=6 * 2.0**-24, atol=1e-44)
    assert all(float(s) == 1 for s in steps)


def test_layouts():
    import trl_amd

    g = torch.Generator().manual_seed(13)
    w = torch.randn(30, 50, generator=g).to(DEV).t()  # dense, another order
    grad = torch.randn(50, 30, generator=g).to(DEV)    # contiguous: copied into that order
    m, v = torch.zeros_like(w), torch.zeros_like(w)
    before = w.clone()
    trl_amd.adamw_step_([w], [grad], [m], [v], step_counters(1), lr=LR, weight_decay=WD)
    want, want_m, _, update = definition(before, grad, torch.zeros(50, 30), torch.zeros(50, 30), 1)
    check_param(w, before, want, update, torch.float32)
    torch.testing.assert_close(m.double().cpu(), want_m, rtol=6 * 2.0**-24, atol=1e-44)
    one = torch.ones(1, device=DEV).expand(50, 30)  # a broadcast gradient
    trl_amd.adamw_step_([w], [one], [m], [v], step_counters(1, 1.0), lr=LR)
    with pytest.raises(ValueError, match="gaps"):
        x = torch.zeros(10, 20, device=DEV)[:, ::2]
        trl_amd.adamw_step_([x], [torch.zeros_like(x)], [torch.zeros(10, 10, device=DEV)], [torch.zeros(10, 10, device=DEV)], step_counters(1))


def test_refusals():
    import trl_amd

    def call(p=None, g=None, m=None, v=None, s=None, **kw):
        x = lambda t=torch.float32, n=600: torch.zeros(n, dtype=t, device=DEV)  # noqa: E731
        return trl_amd.adamw_step_([x()] if p is None else p, [x()] if g is None else g, [x()] if m is None else m,
                                   [x()] if v is None else v, step_counters(1) if s is None else s, **kw)

    call()
    x = torch.zeros(600, device=DEV)
    for kw, error in ((dict(g=[x.bfloat16()]), TypeError), (dict(g=[x[:5]]), ValueError), (dict(m=[x.bfloat16()]), TypeError),
                      (dict(v=[x.byte()]), TypeError), (dict(s=[x]), ValueError), (dict(s=step_counters(2)), ValueError),
                      (dict(p=[x.double()], g=[x.double()]), TypeError), (dict(p=[]), (ValueError, NotImplementedError)),
                      (dict(g=[x.cpu()]), RuntimeError), (dict(s=[torch.zeros(())]), RuntimeError), (dict(lr=-1.0), ValueError),
                      (dict(betas=(1.0, 0.9)), ValueError), (dict(eps=-1.0), ValueError), (dict(weight_decay=-1.0), ValueError),
                      (dict(max_grad_norm=-1.0), ValueError), (dict(max_grad_norm=math.nan), ValueError), (dict(lr=x), ValueError)):
        with pytest.raises(error):
            call(**kw)
    y = torch.zeros(600, device=DEV)
    with pytest.raises(ValueError, match="twice"):
        call([x, x], [y, y], [y.clone(), y.clone()], [y.clone(), y.clone()], step_counters(2))
    with pytest.raises(ValueError, match="twice"):
        call([x, y], [y, y], [y.clone(), y.clone()], [y.clone(), y.clone()], step_counters(1) * 2)
    code = torch.zeros(600, dtype=torch.uint8, device=DEV)
    with pytest.raises(ValueError, match="scales"):
        call([x], [y], [code.view(torch.float8_e4m3fn)], [code.clone()])
    s = torch.ones(2, device=DEV)
    with pytest.raises(ValueError, match="scales"):
        call([x], [y], [code.view(torch.float8_e4m3fn)], [code.clone()], exp_avg_scales=[s], exp_avg_sq_scales=[s])
    with pytest.raises((RuntimeError, NotImplementedError)):
        z = torch.zeros(5)
        trl_amd.adamw_step_([z], [z.clone()], [z.clone()], [z.clone()], [torch.zeros(())])
    with pytest.raises(ValueError):
        trl_amd.adamw_state_values(code, s)
    with pytest.raises(TypeError):
        trl_amd.adamw_state_values(x, torch.ones(3, device=DEV))
    for kw in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(state_bits=16), dict(max_grad_norm=-1.0)):
        with pytest.raises(ValueError):
            trl_amd.AdamW([torch.zeros(3, device=DEV, requires_grad=True)], **kw)


def test_a_saved_parameter_that_has_changed_is_noticed():
    import trl_amd

    w = torch.randn(40, device=DEV, requires_grad=True)
    loss = (w * w).sum()
    w.grad = torch.ones_like(w)
    trl_amd.AdamW([w]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


# ---- the optimiser ----------------------------------------------------------------------------------------------------
def small_model(seed, dtype=torch.float32):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Embedding(97, 64), torch.nn.Linear(64, 130), torch.nn.GELU(), torch.nn.Linear(130, 97)).to(DEV, dtype)


def groups_of(model):
    decay = [p for p in model.parameters() if p.dim() > 1]
    rest = [p for p in model.parameters() if p.dim() <= 1]
    return [dict(params=decay, weight_decay=0.05), dict(params=rest, weight_decay=0.0, lr=3e-3)]


def test_optimiser_follows_torch():
    """20 steps with two groups and clipping, beside torch's optimiser in 64 bits on the same gradients.  An entry's fp32 arithmetic
    drifts by at most 2e-6 of each step's update (of size lr), and 2^-24 of the parameter twice."""
    import trl_amd

    model, double = small_model(1), small_model(1).double()
    double.load_state_dict(model.state_dict())
    ours = trl_amd.AdamW(groups_of(model), lr=1e-2, betas=(0.9, 0.99), max_grad_norm=0.5)
    theirs = torch.optim.AdamW(groups_of(double), lr=1e-2, betas=(0.9, 0.99), foreach=False)
    g = torch.Generator().manual_seed(2)
    for i in range(20):
        for a, b in zip(model.parameters(), double.parameters()):
            x = torch.randn(a.shape, generator=g).to(DEV)
            a.grad, b.grad = x, x.double()
        if i == 3:
            list(model.parameters())[1].grad = list(double.parameters())[1].grad = None
        ours.step()
        norm = torch.nn.utils.clip_grad_norm_(double.parameters(), 0.5)
        theirs.step()
        assert abs(float(ours.grad_norm) / float(norm) - 1) < 2.0**-23
    for a, b in zip(model.parameters(), double.parameters()):
        off = (a.detach().double() - b.detach()).abs()
        assert bool((off <= 20 * (2e-6 * 1e-2 * 3 + 2.0**-23 * b.detach().abs())).all()), off.max()


def test_state_dict_keeps_types():
    import trl_amd

    for bits in (8, 32):
        model, other = small_model(3, torch.bfloat16), small_model(3, torch.bfloat16)
        a, b = (trl_amd.AdamW(groups_of(x), lr=1e-3, state_bits=bits, max_grad_norm=1.0, seed=4) for x in (model, other))
        g = torch.Generator().manual_seed(5)

        def grads(m):
            for p in m.parameters():
                p.grad = torch.randn(p.shape, generator=g).to(DEV, torch.bfloat16)

        for _ in range(2):
            grads(model)
            a.step()
        kinds = {p.numel() >= 4096: s["exp_avg"].dtype for p, s in a.state.items()}
        assert kinds == {True: torch.float8_e4m3fn if bits == 8 else torch.float32, False: torch.float32}
        other.load_state_dict(model.state_dict())
        b.load_state_dict(a.state_dict())
        for p, q in zip(model.parameters(), other.parameters()):
            for k, x in a.state[p].items():
                y = b.state[q][k]
                assert x.dtype == y.dtype and x.data_ptr() != y.data_ptr()
        grads(model)
        for p, q in zip(model.parameters(), other.parameters()):
            q.grad = p.grad.clone()
        a.step()
        b.step()
        for p, q in zip(model.parameters(), other.parameters()):
            assert torch.equal(p, q) and all(torch.equal(x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x,
                                                         b.state[q][k].view(torch.uint8) if x.dtype == torch.float8_e4m3fn else b.state[q][k])
                                             for k, x in a.state[p].items())


def test_a_captured_step_counts():
    """A step in a graph, with its learning rate on the GPU: four replays against four eager steps, bit for bit, on another stream too."""
    import trl_amd

    for bits in (32, 8):
        g = torch.Generator().manual_seed(17)
        w = [torch.randn(s, generator=g).to(DEV) for s in ((300, 41), (5000,), (7,))]
        eager, captured = ([torch.nn.Parameter(x.clone()) for x in w] for _ in range(2))
        lr = torch.tensor(1e-2, device=DEV)
        a = trl_amd.AdamW(eager, lr=lr, state_bits=bits, max_grad_norm=1.0)
        b = trl_amd.AdamW(captured, lr=lr, state_bits=bits, max_grad_norm=1.0)
        for p in captured:
            p.grad = torch.zeros_like(p)
            b._state_of(p, b.param_groups[0])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            b.step()
        for i in range(4):
            lr.fill_(1e-2 / (i + 1))
            for p, q in zip(eager, captured):
                x = torch.randn(p.shape, generator=g).to(DEV)
                p.grad = x
                q.grad.copy_(x)
            graph.replay()
            torch.cuda.synchronize()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                a.step()
            torch.cuda.current_stream().wait_stream(side)
            for p, q in zip(eager, captured):
                assert torch.equal(p, q) and float(a.state[p]["step"]) == float(b.state[q]["step"]) == i + 1
            assert torch.equal(a.grad_norm, b.grad_norm)


def test_one_on_policy_step_end_to_end():
    """Tokens drawn from a small model under top-k and top-p, scored under the distribution they were drawn from, a policy
    gradient through that score, the step: log-probs of drawing and scoring agree, the gradient is the definition's, and the
    parameters move as the optimiser's definition says."""
    import trl_amd

    model = small_model(6)
    s = dict(temperature=0.8, top_k=20, top_p=0.9)
    g = torch.Generator().manual_seed(7)
    prompt = torch.randint(0, 97, (16,), generator=g).to(DEV)
    advantages = torch.randn(16, generator=g).to(DEV)
    opt = trl_amd.AdamW(model.parameters(), lr=1e-2, weight_decay=0.1, max_grad_norm=0.1)
    with torch.no_grad():
        ids, sampled = trl_amd.sample_tokens(model(prompt), torch.rand(16, generator=g).to(DEV), **s)
    logits = model(prompt)
    logps = trl_amd.filtered_logps(logits, ids, **s)
    assert torch.equal(logps.detach(), sampled)
    loss = -(torch.exp(logps - sampled) * advantages).mean()
    loss.backward()
    # the same gradient in 64 bits, from a softmax over the kept tokens
    twin = small_model(6).double()
    z = twin(prompt) / s["temperature"]
    order = z.argsort(dim=-1, descending=True)[:, :20]
    top = z.gather(1, order).softmax(-1)
    keep = top.cumsum(-1) - top < s["top_p"]
    mask = torch.zeros_like(z, dtype=torch.bool).scatter_(1, order, keep)
    want = z.masked_fill(~mask, -math.inf).log_softmax(-1).gather(1, ids[:, None]).squeeze(1)
    (-(torch.exp(want - want.detach()) * advantages.double()).mean()).backward()
    for p, q in zip(model.parameters(), twin.parameters()):
        # (fp32 products over at most 130 entries and 16 rows: a few hundred roundings of 2^-24)
        assert float((p.grad.double() - q.grad).norm()) <= 1e-4 * float(q.grad.norm())
    before = [p.detach().clone() for p in model.parameters()]
    norm = norm64([p.grad for p in model.parameters()])
    opt.step()
    trl_amd.check_device_errors()
    assert abs(float(opt.grad_norm) / norm - 1) < 2.0**-23
    for x, p in zip(before, model.parameters()):
        zero = torch.zeros(p.shape)
        want_p, _, _, update = definition(x, p.grad, zero, zero, 1, min(1.0, 0.1 / (norm + 1e-6)), lr=1e-2, wd=0.1)
        check_param(p.detach(), x, want_p, update, torch.float32, lr=1e-2)


def test_traced_calls_have_the_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import trl_amd

    with FakeTensorMode():
        x = [torch.empty(300, device=DEV, dtype=torch.bfloat16), torch.empty(7, 5, device=DEV, dtype=torch.bfloat16)]
        m = [torch.empty(t.shape, device=DEV) for t in x]
        steps = [torch.empty((), device=DEV) for _ in x]
        norm = trl_amd.adamw_step_(x, [t.clone() for t in x], m, [t.clone() for t in m], steps, max_grad_norm=1.0)
        assert norm.shape == () and norm.dtype == torch.float32 and norm.device.type == "cuda"
        assert trl_amd.adamw_step_(x, [t.clone() for t in x], m, [t.clone() for t in m], steps) is None
        values = trl_amd.adamw_state_values(torch.empty(600, device=DEV, dtype=torch.uint8), torch.empty(3, device=DEV))
        assert values.shape == (600,) and values.dtype == torch.bfloat16


def test_one_learning_rate_for_each_group_and_empty_tensors():
    """Groups with rates on the host and on the GPU, tensors of no and of one entry, and one without a gradient, against torch's AdamW."""
    import trl_amd

    g = torch.Generator().manual_seed(71)
    shapes = ((0,), (1,), (4097,), (3, 0, 2), (70, 71), (5,))
    mine, theirs = ([torch.nn.Parameter(torch.randn(s, generator=torch.Generator().manual_seed(i)).to(DEV)) for i, s in enumerate(shapes)]
                    for _ in range(2))
    groups = lambda w, lr: [dict(params=w[:2], lr=1e-2), dict(params=w[2:5], lr=lr, weight_decay=0.1), dict(params=w[5:], eps=1e-3)]  # noqa: E731
    a = trl_amd.AdamW(groups(mine, torch.tensor(3e-3, device=DEV)), lr=1e-3)
    b = torch.optim.AdamW(groups(theirs, 3e-3), lr=1e-3, foreach=False)
    for _ in range(4):
        for p, q in zip(mine[:5], theirs[:5]):
            p.grad = torch.randn(p.shape, generator=g).to(DEV)
            q.grad = p.grad.clone()
        a.step()
        b.step()
    for p, q in zip(mine, theirs):
        # four steps, each a few roundings of a step of 1e-2 at most and one of the value
        assert torch.allclose(p, q, rtol=4 * 2.0**-23, atol=4 * 1e-2 * 8 * 2.0**-24)
    assert mine[5].grad is None and not a.state.get(mine[5])


# ---- tiny second moments ----------------------------------------------------------------------------------------------
TINY = [0.0, 1e-24, 2e-23, 1.5e-22, 1e-21, 3e-20, 1e-19, 2e-18, 1e-15, 1e-8, 1.0]  # (g^2 (1 - b2) is 0, subnormal up to 3e-18, normal)


def tiny_step(bits, eps, t, seed=0):
    """One step from zero moments on gradients of these sizes: parameters, moments (in 64 bits, from their fp32 arithmetic), results."""
    import trl_amd

    g = torch.tensor(TINY, dtype=torch.float64).float().repeat_interleave(256) * torch.tensor([1.0, -1.0]).repeat(len(TINY) * 128)
    p = torch.randn(g.numel(), generator=torch.Generator().manual_seed(seed))
    w, grad = p.to(DEV, t), g.to(DEV, t)
    g, p = grad.cpu().float(), w.cpu()
    if bits == 32:
        m, v = [torch.zeros(g.numel(), device=DEV)], [torch.zeros(g.numel(), device=DEV)]
        kw = {}
    else:
        m, v, ms, vs = eight_bit_state([(g.numel(),)])
        kw = dict(exp_avg_scales=ms, exp_avg_sq_scales=vs)
    trl_amd.adamw_step_([w], [grad], m, v, step_counters(1), lr=LR, betas=(B1, B2), eps=eps, weight_decay=WD, **kw)
    one_minus_b1, one_minus_b2 = torch.tensor(1 - B1).float(), torch.tensor(1 - B2).float()
    return w, p, (g * one_minus_b1).double(), (g * g * one_minus_b2).double(), m, v


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [0.0, 2.0**-130, 1e-30, 1e-21, 1e-12, 1e-8])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_tiny_second_moments(bits, eps, dtype):
    """Second moments that are subnormal, and an eps that does not hide them: the update is the formula's.  Its root and reciprocal are off by
    a unit of 2^-23 each, scaling by powers of two is exact, so the bounds are those of `check_param`; eps and a sum with it are normal
    numbers, or exact."""
    t = DTYPES[dtype]
    w, p, m, v, got_m, got_v = tiny_step(bits, eps, t)
    if bits == 32:
        assert torch.equal(got_m[0].cpu().double(), m) and torch.equal(got_v[0].cpu().double(), v)
        assert int(((v > 0) & (v < 2.0**-126)).sum()) >= 4 * 256 and int((v == 0).sum()) >= 2 * 256
    eps32 = float(torch.tensor(eps).float())
    update = (m / (1 - B1)) / ((v / (1 - B2)).sqrt() + eps32)
    want = p.double() * (1 - LR * WD) - LR * update
    finite = want.abs() < torch.finfo(t).max / 2
    check_param(w.cpu()[finite], p[finite], want[finite], update[finite], t)
    rest = w.cpu()[~finite].double()
    # (0 / 0 is a NaN, anything else over 0 infinite, as in `torch.optim.AdamW`; what is too large for the type is infinite, too)
    assert torch.equal(rest.isnan(), want[~finite].isnan()) and bool((rest.isnan() | (rest.abs() >= torch.finfo(t).max / 4)).all())
    assert bool(finite.all()) == (eps > 0)


def test_a_profiler_sees_the_operator():
    import trl_amd

    p, grads, put = make([(300,)], torch.float32, 3)
    m, v = zeros32([(300,)], put)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        trl_amd.adamw_step_(p, grads, m, v, step_counters(1))
    assert "trl_amd::adamw_step_" in {e.key for e in prof.key_averages()}
