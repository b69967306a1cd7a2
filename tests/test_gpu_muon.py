"""Orthogonalised updates (`orthogonalize`, `muon_step_`, `Muon`) against their definition in 64 bits.

Tolerances (2-norms of whole matrices).  16 bits: the iteration rounds the products' operands to fp16; `rounded` makes the same roundings at the
same places in 64 bits, and how far that is from the exact iteration is what the formats cost for a given matrix.  Kernels sum in fp32 and round to
other neighbours here and there: 1.5 times that, and half a step of the output's type.  fp32, and results in fp16: the operands hold 22 bits and sums are
fp32, as in an iteration in plain fp32, whose own distance from the exact one on the same matrix is taken 4 times (a product of two pieces drops
2^-22, four times fp32's rounding), and 1e-6.  Momentum: three roundings of 2^-24 of the summands.  Parameters: two roundings of fp32 and
half a step of their type beside the update's error."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
A, B, C = 3.4445, -4.7750, 2.0315
SHAPES = [(1, 1), (1, 7), (7, 1), (5, 5), (16, 500), (500, 16), (63, 65), (64, 64), (65, 64), (100, 1), (13, 2050), (129, 300), (300, 129),
          (256, 256), (257, 513), (640, 1001), (1001, 321), (520, 520)]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def exact(u, steps=5, coefficients=(A, B, C), eps=1e-7):
    a, b, c = coefficients
    x = u.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / max(float(torch.linalg.vector_norm(x)), eps)
    for _ in range(steps):
        gram = x @ x.mT
        x = a * x + (b * gram + c * gram @ gram) @ x
    return x.mT if tall else x


def fp16(x, unit):
    return (x * unit).to(torch.float16).double() / unit


def rounded(u, steps=5, coefficients=(A, B, C), eps=1e-7):
    """The iteration in 64 bits with its operands rounded as the kernels round them."""
    a, b, c = coefficients
    x = u.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / max(float(torch.linalg.vector_norm(x)), eps)
    for step in range(steps):
        hi = fp16(x, 16384.0)
        x = hi + fp16(x - hi, 16384.0) if step == 0 or step + 1 < steps else hi
        gram = fp16(hi @ hi.mT, 8192.0)
        factor = b * gram + c * gram @ gram
        x = a * x + fp16(factor, 8192.0) @ hi + torch.diag(factor - fp16(factor, 8192.0))[:, None] * hi  # (B's diagonal loses nothing)
    return x.mT if tall else x


def plain32(u, steps=5, coefficients=(A, B, C), eps=1e-7):
    a, b, c = coefficients
    x = u.float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT.contiguous() if tall else x
    x = x / max(float(torch.linalg.vector_norm(x.double())), eps)
    for _ in range(steps):
        gram = x @ x.mT.contiguous()
        x = a * x + (b * gram + c * gram @ gram) @ x
    return x.mT if tall else x


def distance(x, y):
    return float(torch.linalg.vector_norm(x.double() - y.double()))


def allowed(u, dtype, want, step=False, **numbers):
    if dtype == torch.float32 or (dtype == torch.float16 and not step):
        return 4 * distance(plain32(u, **numbers), want) + 1e-6 * float(want.norm())
    return 1.5 * distance(rounded(u, **numbers), want) + 1e-6 * float(want.norm())


def check(got, u, **numbers):
    want = exact(u, **numbers)
    bound = allowed(u, got.dtype, want, **numbers) + half_step(got.dtype) * float(want.norm()) + 1e-30
    assert got.shape == u.shape and distance(got, want) <= bound, (distance(got, want), bound, float(want.norm()))


def spectrum(shape, kind, gen):
    x = torch.randn(shape, generator=gen, device=DEV)
    if kind == "even":
        return x
    r = min(shape)
    u, _, v = torch.linalg.svd(x.cpu(), full_matrices=False)
    i = torch.arange(1, r + 1)
    s = {"falling": i**-1.0, "steep": torch.exp(-i / max(1.0, r / 8)), "few": (i <= max(1, r // 16)) + 1e-6}[kind]
    return ((u * s) @ v).to(DEV)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(dtype, shape):
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(shape[0] * 7 + shape[1])
    for kind, size in (("even", 1.0), ("even", 1e-4), ("falling", 30.0), ("steep", 1.0), ("few", 1.0)):
        u = (spectrum(shape, kind, gen) * size).to(DTYPES[dtype])
        got = trl_amd.orthogonalize(u)
        assert got.dtype == u.dtype
        check(got, u)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_many_matrices_in_one_call(dtype):
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(3)
    shapes = [s for s in SHAPES if max(s) < 600] * 2 + [(3, 70, 40), (2, 2, 33, 90), (0, 4, 4), (4, 0), (0, 4), (2, 0, 3)]
    each = [torch.randn(s, generator=gen, device=DEV).to(DTYPES[dtype]) for s in shapes]
    each += [torch.randn((90, 200), generator=gen, device=DEV).to(DTYPES[dtype]).t()]  # another order of entries
    got = trl_amd.orthogonalize(each)
    assert len(got) == len(each)
    for u, x in zip(each, got):
        assert x.shape == u.shape
        for um, xm in zip(u.reshape(-1, *u.shape[-2:]) if u.numel() else [], x.reshape(-1, *u.shape[-2:]) if u.numel() else []):
            check(xm, um)
            assert torch.equal(xm, trl_amd.orthogonalize(um))  # alone or among others: the same bits
    mixed = trl_amd.orthogonalize([each[0].float(), each[3].bfloat16(), each[4].half()])
    assert [x.dtype for x in mixed] == [torch.float32, torch.bfloat16, torch.float16]
    assert trl_amd.orthogonalize([]) == []


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shapes", [[(1703, 1801)] * 5 + [(1801, 1703)] * 4, [(1150, 700), (700, 1150), (2100, 90), (90, 2100), (900, 900)]])
def test_larger_matrices(dtype, shapes):
    """Launches of as many 256 x 256 tiles as there are CUs, and of few."""
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(4)
    each = [(torch.randn((s[0], 200), generator=gen, device=DEV) @ torch.randn((200, s[1]), generator=gen, device=DEV) * 0.3 + torch.randn(s, generator=gen, device=DEV)).to(DTYPES[dtype])
            for s in shapes]
    for u, x in zip(each, trl_amd.orthogonalize(each)):
        check(x, u)


@pytest.mark.parametrize("shape", [(1100, 1 << 22), (1 << 22, 1100)])
def test_offsets_past_32_bits(shape):
    """With G = X X^T in 64 bits the result is T X, T the product of the steps' factors: columns from all over the matrix.  The bound: operands of 11
    bits cost independent entries 1.7e-3 of the result at most (`rounded` on such matrices), and the rounding to bf16 half a step."""
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(6)
    u = torch.empty(shape, dtype=torch.bfloat16, device=DEV)
    for part in u.view(-1).split(1 << 28):
        part.normal_(generator=gen)
    x = u if shape[0] < shape[1] else u.t()
    rows, cols = x.shape
    gram = torch.zeros((rows, rows), dtype=torch.float64, device=DEV)
    for c in range(0, cols, 1 << 17):
        part = x[:, c : c + (1 << 17)].double()
        gram += part @ part.t().contiguous()
    factor = 1 / gram.trace().sqrt()
    gram *= factor**2
    steps, eye = torch.eye(rows, dtype=torch.float64, device=DEV), torch.eye(rows, dtype=torch.float64, device=DEV)
    for _ in range(5):
        p = A * eye + B * gram + C * gram @ gram
        steps, gram = p @ steps, p @ gram @ p
    got = trl_amd.orthogonalize(u)
    got = got if shape[0] < shape[1] else got.t()
    for c in (0, cols // 2 - 777, cols - 4096):
        want = steps @ (x[:, c : c + 4096].double() * factor)
        assert distance(got[:, c : c + 4096], want) <= (1.5 * 1.7e-3 + 2.0**-8) * float(want.norm())


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_other_numbers(dtype):
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(5)
    for shape in ((70, 30), (90, 333)):
        u = torch.randn(shape, generator=gen, device=DEV).to(DTYPES[dtype])
        for steps, coefficients in ((1, (A, B, C)), (2, (1.5, -0.5, 0.0)), (8, (2.0, -1.5, 0.5)), (3, (1.875, -1.25, 0.375)), (1, (1.0, 0.0, 0.0))):
            got = trl_amd.orthogonalize(u, ns_coefficients=coefficients, ns_steps=steps)
            check(got, u, steps=steps, coefficients=coefficients)


def test_degenerate_matrices():
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(6)
    for t in DTYPES.values():
        for shape in ((40, 70), (300, 270)):
            zero, fine = torch.zeros(shape, dtype=t, device=DEV), torch.randn(shape, generator=gen, device=DEV).to(t)
            nan, inf = fine.clone(), fine.clone()
            nan[3, 5], inf[-1, -1] = math.nan, math.inf
            a, b, c, d = trl_amd.orthogonalize([zero, nan, fine, inf])
            assert not a.any() and bool(b.isnan().all()) and bool(d.isnan().all())
            check(c, fine)
            same = torch.ones(shape, dtype=t, device=DEV)  # rank one
            check(trl_amd.orthogonalize(same), same)
    # sizes at both ends of fp32's range, and norms below eps: the iteration stretches those by 3.4445^5 = 485.  X is held in units of 2^-14 in two
    # pieces of fp16, the lower one a multiple of 2^-24: rounded by 2^-39 at the start, and half a step and 2^-39 times the stretch in each of five iterations
    u = torch.randn((50, 60), generator=gen, device=DEV)
    for size in (1e-30, 1e18):
        got, want = trl_amd.orthogonalize(u * size, eps=1e-7 if size > 1 else 1e-7), exact(u * size)
        assert distance(got, want) <= 4 * distance(plain32(u * size), want) + 1e-6 * float(want.norm()) + 5 * 485 * 2.0**-38 * math.sqrt(3000)
    for size in (1e-9, 1e-11):
        got, want = trl_amd.orthogonalize(u * size), exact(u * size)
        assert distance(got, want) <= 1e-5 * float(want.norm()) + 5 * 485 * 2.0**-38 * math.sqrt(3000)


def make(shapes, dtype, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    p = [torch.randn(s, generator=gen, device=DEV).mul_(0.05).to(dtype) for s in shapes]
    g = [torch.randn(s, generator=gen, device=DEV).mul_(1e-3).to(dtype) for s in shapes]
    m = [torch.randn(s, generator=gen, device=DEV).mul_(1e-3) for s in shapes]
    return p, g, m


def definition(p, g, m, lr, wd, beta, nesterov, adjust, **numbers):
    """(parameter, momentum, the 2-norm that the update may be off by) of one matrix, in 64 bits."""
    g, m = g.double(), m.double()
    now = beta * m + (1 - beta) * g
    u = beta * now + (1 - beta) * g if nesterov else now
    rows, cols = p.shape
    stretch = 0.2 * math.sqrt(max(rows, cols)) if adjust == "match_rms_adamw" else math.sqrt(max(1.0, rows / cols))
    x = exact(u, **numbers)
    off = lr * stretch * allowed(u.float(), p.dtype, x, step=True, **numbers)
    return p.double() * (1 - lr * wd) - lr * stretch * x, now, off


def check_step(p, m, before_p, before_g, before_m, **settings):
    for i in range(len(p)):
        shape = p[i].shape[-2:]
        for now_p, now_m, was_p, g, was_m in zip(*(t.reshape(-1, *shape) for t in (p[i], m[i], before_p[i], before_g[i], before_m[i]))):
            want_p, want_m, off = definition(was_p, g, was_m, **settings)
            beta = settings["beta"]
            sizes = beta * was_m.double().abs() + (1 - beta) * g.double().abs()
            assert bool(((now_m.double() - want_m).abs() <= 4 * 2.0**-24 * sizes).all())
            assert distance(now_p, want_p) <= off + (2.0**-23 + half_step(p[i].dtype)) * (float(want_p.norm()) + float(was_p.double().norm()))


STEP_SHAPES = [(16, 200), (200, 16), (70, 70), (130, 290), (290, 130), (3, 65, 40), (1, 9)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("settings", [dict(lr=0.02, wd=0.1, beta=0.95, nesterov=True, adjust=None),
                                      dict(lr=1e-3, wd=0.0, beta=0.9, nesterov=False, adjust="match_rms_adamw"),
                                      dict(lr=0.5, wd=1.0, beta=0.0, nesterov=True, adjust="original")])
def test_step(dtype, settings):
    import trl_amd

    p, g, m = make(STEP_SHAPES, DTYPES[dtype], 8)
    for _ in range(2):
        before = [[t.clone() for t in x] for x in (p, g, m)]
        trl_amd.muon_step_(p, g, m, lr=settings["lr"], weight_decay=settings["wd"], momentum=settings["beta"], nesterov=settings["nesterov"],
                           adjust_lr_fn=settings["adjust"])
        assert all(torch.equal(x, y) for x, y in zip(g, before[1]))
        check_step(p, m, *before, **settings)
    # the same call gives the same bits, with a learning rate on the GPU too, and with gradients in another order
    q, k = [t.clone() for t in before[0]], [t.clone() for t in before[2]]
    other = [t.mT.contiguous().mT for t in g]
    trl_amd.muon_step_(q, other, k, lr=torch.tensor(settings["lr"], device=DEV), weight_decay=settings["wd"], momentum=settings["beta"],
                       nesterov=settings["nesterov"], adjust_lr_fn=settings["adjust"])
    assert all(torch.equal(x, y) for x, y in zip(k, m))
    if DTYPES[dtype] != torch.float32:  # (a number and its fp32 value may differ in fp32's last place)
        assert sum(int((x != y).sum()) for x, y in zip(q, p)) <= 0.001 * sum(x.numel() for x in p)
    assert all(distance(x, y) <= 2.0**-22 * float(x.double().norm()) + half_step(x.dtype) * float(x.double().norm()) for x, y in zip(q, p))


def test_groups_of_the_optimizer_and_the_rest():
    import trl_amd

    torch.manual_seed(0)
    shapes = [(48, 96), (96, 48), (40, 40)]
    w = [torch.nn.Parameter(torch.randn(s, device=DEV) * 0.05) for s in shapes]
    rest = [torch.nn.Parameter(torch.randn(s, device=DEV)) for s in ((96,), (97, 48))]
    idle = torch.nn.Parameter(torch.randn((5, 5), device=DEV))
    lr_gpu = torch.tensor(0.01, device=DEV)
    opt = trl_amd.Muon([dict(params=w[:2] + [idle]), dict(params=w[2:], lr=lr_gpu, momentum=0.5, nesterov=False, weight_decay=0.0, ns_steps=3,
                                                          adjust_lr_fn="match_rms_adamw"), dict(params=rest, adamw=True, lr=1e-2, betas=(0.8, 0.9))],
                       lr=0.02, weight_decay=0.05)
    reference = torch.optim.AdamW([r.detach().clone().requires_grad_(True) for r in rest], lr=1e-2, betas=(0.8, 0.9), weight_decay=0.05)
    twins = reference.param_groups[0]["params"]
    for step in range(3):
        for p in w + rest:
            p.grad = torch.randn_like(p) * 1e-2
        for t, r in zip(twins, rest):
            t.grad = r.grad.clone()
        before = [[p.detach().clone() for p in w], [p.grad.clone() for p in w],
                  [opt.state[p]["momentum_buffer"].clone() if step else torch.zeros_like(p) for p in w]]
        assert opt.step() is None
        reference.step()
        momenta = [opt.state[p]["momentum_buffer"] for p in w]
        check_step([p.detach() for p in w[:2]], momenta[:2], *(x[:2] for x in before), lr=0.02, wd=0.05, beta=0.95, nesterov=True, adjust=None)
        check_step([w[2].detach()], momenta[2:], *(x[2:] for x in before), lr=float(lr_gpu), wd=0.0, beta=0.5, nesterov=False,
                   adjust="match_rms_adamw", steps=3)
        for t, r in zip(twins, rest):
            torch.testing.assert_close(r, t, rtol=1e-5, atol=1e-6)
    assert idle not in opt.state or not opt.state[idle]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_state_goes_on(dtype):
    """A run that is stopped, saved and taken up is the run that was not; torch's own state is taken."""
    import copy

    import trl_amd

    def model():
        torch.manual_seed(1)
        p = [torch.nn.Parameter((torch.randn(s, device=DEV) * 0.1).to(DTYPES[dtype])) for s in ((30, 50), (80, 20), (7,))]
        return p, trl_amd.Muon([dict(params=p[:2]), dict(params=p[2:], adamw=True)], lr=0.01)

    def steps(p, opt, seeds):
        for s in seeds:
            gen = torch.Generator(device=DEV).manual_seed(s)
            for x in p:
                x.grad = torch.randn(x.shape, generator=gen, device=DEV).to(x.dtype)
            opt.step()

    p, opt = model()
    steps(p, opt, range(4))
    q, other = model()
    steps(q, other, range(2))
    saved = copy.deepcopy(other.state_dict())
    r, again = model()
    with torch.no_grad():
        for x, y in zip(r, q):
            x.copy_(y)
    again.load_state_dict(saved)
    assert all(again.state[x]["momentum_buffer"].dtype == torch.float32 for x in r[:2])
    steps(r, again, range(2, 4))
    assert all(torch.equal(x, y) for x, y in zip(p, r))
    theirs = torch.optim.Muon([x.detach().clone().requires_grad_(True) for x in p[:2]], lr=0.01)
    for x in theirs.param_groups[0]["params"]:
        x.grad = torch.randn_like(x)
    theirs.step()
    mine = trl_amd.Muon([x.detach().clone().requires_grad_(True) for x in p[:2]], lr=0.5)
    mine.load_state_dict(theirs.state_dict())
    assert mine.param_groups[0]["lr"] == 0.01
    for x, y in zip(mine.param_groups[0]["params"], theirs.param_groups[0]["params"]):
        assert torch.equal(mine.state[x]["momentum_buffer"], theirs.state[y]["momentum_buffer"].float())
        x.grad = torch.randn_like(x)
    mine.step()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_graph_capture(dtype):
    import trl_amd

    p, g, m = make(STEP_SHAPES, DTYPES[dtype], 11)
    lr = torch.tensor(0.02, device=DEV)
    step = lambda: trl_amd.muon_step_(p, g, m, lr=lr)  # noqa: E731
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    gen = torch.Generator(device=DEV).manual_seed(1)
    for i in range(4):
        for x in g:
            x.copy_(torch.randn(x.shape, generator=gen, device=DEV) * 1e-3)
        lr.fill_(0.01 * (i + 1))
        q, k = [x.clone() for x in p], [x.clone() for x in m]
        graph.replay()
        torch.cuda.synchronize()
        trl_amd.muon_step_(q, g, k, lr=lr)
        assert all(torch.equal(x, y) for x, y in zip(p + m, q + k))


def test_through_the_operator_or_past_it():
    """A dispatch mode sees the operator; tuples are no lists of plain tensors.  The results are the same to the last bit."""
    from torch.utils._python_dispatch import TorchDispatchMode

    import trl_amd

    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    lr = torch.tensor(0.1, device=DEV)
    results = []
    for way in ("past", "mode", "tuples"):
        p, g, m = make([(20, 30), (90, 80), (0, 3)], torch.bfloat16, 4)
        if way == "mode":
            with Watch():
                trl_amd.muon_step_(p, g, m, lr=lr)
        else:
            trl_amd.muon_step_(p if way == "past" else tuple(p), g, m, lr=lr)
        results.append(p + m)
    assert any("muon_step_" in name for name in seen)
    for other in results[1:]:
        assert all(torch.equal(x, y) for x, y in zip(results[0], other))


def test_versions_and_inference_tensors():
    import trl_amd

    p, g, m = make([(20, 30)], torch.float32, 2)
    version = p[0]._version, m[0]._version
    trl_amd.muon_step_(p, g, m)
    assert p[0]._version > version[0] and m[0]._version > version[1]
    with torch.inference_mode():
        q = [x.clone() for x in p]
        trl_amd.muon_step_(q, [x.clone() for x in g], [x.clone() for x in m])
    x = torch.randn((4, 5), device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError):
        trl_amd.orthogonalize(x).sum().backward()


def test_refusals():
    import trl_amd

    p, g, m = make([(20, 30), (30, 20)], torch.float32, 2)
    good = dict(params=p, grads=g, momentum_buffers=m)

    def call(**changed):
        a = {**good, **changed}
        trl_amd.muon_step_(a["params"], a["grads"], a["momentum_buffers"], **{k: v for k, v in a.items() if k not in good})

    kept = [x.clone() for x in p + m]
    for changed in (dict(grads=g[:1]), dict(grads=[g[1], g[0]]), dict(momentum_buffers=[p[0], m[1]]), dict(params=[p[0], p[0]], grads=[g[0], g[0]], momentum_buffers=[m[0], m[0].clone()]),
                    dict(grads=[p[0], g[1]]), dict(params=[p[0].t(), p[1].t()], grads=[x.t() for x in g], momentum_buffers=[x.t() for x in m]),
                    dict(params=[], grads=[], momentum_buffers=[]), dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(adjust_lr_fn="other"),
                    dict(ns_steps=0), dict(ns_steps=101), dict(eps=0.0), dict(ns_coefficients=(1.0, 2.0)), dict(ns_coefficients=(9.0, 0.0, 0.0)),
                    dict(ns_coefficients=(math.nan, 0.0, 0.0)), dict(params=[x[0] for x in p], grads=[x[0] for x in g], momentum_buffers=[x[0] for x in m])):
        with pytest.raises(ValueError):
            call(**changed)
    for changed in (dict(grads=[x.half() for x in g]), dict(momentum_buffers=[x.half() for x in m]),
                    dict(params=[x.double() for x in p], grads=[x.double() for x in g])):
        with pytest.raises(TypeError):
            call(**changed)
    with pytest.raises(RuntimeError):
        call(grads=[x.cpu() for x in g])
    assert all(torch.equal(x, y) for x, y in zip(p + m, kept))
    with pytest.raises(ValueError):
        trl_amd.orthogonalize(torch.randn(5, device=DEV))
    with pytest.raises(TypeError):
        trl_amd.orthogonalize(torch.randn((5, 5), device=DEV, dtype=torch.float64))
    sparse = torch.nn.Parameter(torch.randn((5, 4), device=DEV))
    sparse.grad = torch.sparse_coo_tensor([[0]], torch.ones((1, 4)), (5, 4), device=DEV)
    with pytest.raises(RuntimeError):
        trl_amd.Muon([sparse]).step()
