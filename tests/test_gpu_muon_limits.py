"""Orthogonalised updates at the limits of what is accepted: many steps, other coefficients, matrices whose entries are alike, norms under eps."""
import math

import pytest
import torch

from test_gpu_muon import A, B, C, DEV, DTYPES, distance, exact, half_step, plain32

pytestmark = pytest.mark.gpu


def test_numbers_that_do_not_fit_are_refused():
    """By the operators too, which `Muon.step` calls with a group's settings as they are now."""
    import trl_amd

    x = torch.ones((4, 5), device=DEV)
    m = torch.zeros_like(x)
    for steps in (2**32 + 5, 0, 101):
        with pytest.raises(ValueError):
            trl_amd.ops.orthogonalize([x], [A, B, C], steps, 1e-7)
        with pytest.raises(ValueError):
            trl_amd.ops.muon_step_([x], [x.clone()], [m], [], [0.1, 0.9, 0.0, 1.0, 0.0], [], [A, B, C], steps, 1e-7)
    for group in (2**32, 1, -1):
        with pytest.raises(ValueError):
            trl_amd.ops.muon_step_([x], [x.clone()], [m], [group], [0.1, 0.9, 0.0, 1.0, 0.0], [], [A, B, C], 5, 1e-7)
    assert bool((x == 1).all()) and not m.any()


def largest_value(a=A, b=B, c=C):
    """Of a s + b s^3 + c s^5 for s up to 1.2: where a + 3 b s^2 + 5 c s^4 is zero for the first time, at s = 0.5545, it is 1.2024; its value there, at 1.2024, is 0.95
    and at 1 it is 0.70."""
    t = (-3 * b - math.sqrt(9 * b * b - 20 * a * c)) / (10 * c)
    return math.sqrt(t) * (a + t * (b + c * t))


def low_rank(shape, rank, gen, whole=False):
    draw = (lambda s: torch.randint(-8, 9, s, generator=gen, device=DEV).float()) if whole else (lambda s: torch.randn(s, generator=gen, device=DEV))
    return draw((shape[0], rank)) @ draw((rank, shape[1]))


def exact_of_rank(u, rank, steps, coefficients=(A, B, C), eps=1e-7):
    """By singular values, those behind the rank being zero, not what rounding has left of them."""
    a, b, c = coefficients
    left, s, right = torch.linalg.svd(u.double().cpu(), full_matrices=False)
    s = s / max(float(s.norm()), eps)
    s[rank:] = 0
    for _ in range(steps):
        s = a * s + b * s**3 + c * s**5
    return ((left * s) @ right).to(u.device)


@pytest.mark.parametrize("steps", [5, 12, 17, 18, 20, 30, 100])
@pytest.mark.parametrize("shape", [(1, 9), (16, 500), (40, 70), (64, 900), (900, 48), (33, 40000)])
def test_narrow_matrices_of_low_rank_and_many_steps(shape, steps):
    """64 rows or fewer go by the Gram matrix, whose rounding moves eigenvalues of zero either way.  Whole numbers of rank one are exactly of that rank in every type:
    the result is u / |u| times one number, which 64 bits hold to 1e-12 after five steps and, the usual polynomial's cycle attracting, to 2e-7 after 100.  A direction
    that is not the matrix's own is taken for one of size 2^-23, grows to size one and stays there (0.68 to 1.21): 1.8 2^23 in all, times the 64 2^-53 of
    the matrix that rounding leaves in it is 1e-7.  So 1e-5 has room for both."""
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(shape[0] + steps)
    for dtype in DTYPES.values():
        u = low_rank(shape, 1, gen, whole=True).to(dtype)
        got, want = trl_amd.orthogonalize(u, ns_steps=steps), exact_of_rank(u, 1, steps)
        assert distance(got, want) <= (1e-5 + half_step(dtype)) * float(want.norm()) + 1e-30, dtype
    # of rank four, rounded to fp32: what the rounding adds is at 2^-24, and comes up by itself from 12 steps on.  Then only the size is known.
    u = low_rank(shape, 4, gen)
    got = trl_amd.orthogonalize(u, ns_steps=steps)
    assert float(torch.linalg.matrix_norm(got.double().cpu(), 2)) <= largest_value() * 1.01
    if steps <= 12:
        want = exact(u, steps=steps)
        assert distance(got, want) <= 4 * distance(plain32(u, steps=steps), want) + 1e-6 * float(want.norm())


def alike(kind, gen):
    """Matrices whose entries or singular values are alike: roundings of their pieces go one way and do not average out."""
    if kind == "ones":
        return torch.ones((113, 120), device=DEV)
    if kind == "ones, many columns":
        return torch.ones((383, 4096), device=DEV)
    if kind == "signs":
        return torch.sign(torch.randn((353, 1), generator=gen, device=DEV)) * torch.sign(torch.randn((1, 360), generator=gen, device=DEV))
    if kind == "identity":
        return torch.eye(353, device=DEV)
    if kind == "orthogonal":
        return torch.linalg.qr(torch.randn((353, 353), generator=gen, device=DEV).cpu())[0].contiguous().to(DEV)
    if kind == "hadamard":
        x = torch.ones((1, 1), device=DEV)
        for _ in range(9):
            x = torch.cat([torch.cat([x, x], 1), torch.cat([x, -x], 1)])
        return x[:, :100].contiguous()
    return torch.randn((128, 512), generator=gen, device=DEV)


KINDS = ["ones", "ones, many columns", "signs", "identity", "orthogonal", "hadamard", "even"]
SENSITIVE = [(5, (A, B, C)), (10, (A, B, C)), (20, (A, B, C)), (5, (4.0848, -6.8946, 2.9270)), (7, (4.0848, -6.8946, 2.9270))]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("steps,coefficients", SENSITIVE)
def test_a_result_is_as_near_as_fp32s(dtype, kind, steps, coefficients):
    """Whatever the type: operands of 22 bits, rounded (or a product of their pieces left out) by 2^-22.  In b A + c A A of a step those are two in A = X X^T and its own,
    so six in A A, its own in both products and X's behind them: 8 at most, of the sizes of b A and c A A.  What they make of a singular value grows by the slopes
    of the steps behind; `growth` is the largest growth of all.  And the result's rounding.  (Sizes: the final singular values are 0.68 and more, 8 / 0.68 < 12.)"""
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(steps)
    u = alike(kind, gen).to(DTYPES[dtype])
    got, want = trl_amd.orthogonalize(u, ns_steps=steps, ns_coefficients=coefficients), exact(u, steps=steps, coefficients=coefficients)
    assert distance(got, want) <= (12 * growth(steps, coefficients) * 2.0**-22 + half_step(got.dtype)) * float(want.norm()), distance(got, want) / float(want.norm())


def growth(steps, coefficients):
    """By how much a relative error of one made in b A + c A A of every step, has grown in the result, for the singular value where that is most."""
    a, b, c = coefficients
    s = torch.arange(1, 257, dtype=torch.float64) / 256
    off = torch.zeros_like(s)
    for _ in range(steps):
        t = s * s
        off = (a + 3 * b * t + 5 * c * t * t).abs() * off + (abs(b) * t + abs(c) * t * t) * s
        s = s * (a + t * (b + c * t))
    return float(off.max())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", [(70, 70), (100, 260), (300, 129)])
@pytest.mark.parametrize("steps", [5, 20, 100])
def test_wide_matrices_of_low_rank_and_many_steps(dtype, shape, steps):
    """What rounding adds to a matrix of low rank comes up by itself.  Its singular values stay under the polynomial's largest value on its way, but for
    the rounding of each step and of the result: 2 per cent have room for both."""
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(shape[0] + steps)
    for rank in (1, 4):
        u = low_rank(shape, rank, gen).to(DTYPES[dtype])
        got = trl_amd.orthogonalize(u, ns_steps=steps)
        assert float(torch.linalg.matrix_norm(got.double().cpu(), 2)) <= largest_value() * 1.02


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("steps,coefficients", SENSITIVE + [(1, (A, B, C)), (4, (A, B, C)), (10, (1.875, -1.25, 0.375)), (8, (2.0, -1.5, 0.5))])
def test_a_step_is_off_by_what_the_usual_five_are_at_most(dtype, kind, steps, coefficients):
    """Parameters of zero and a learning rate of one: the step leaves minus the update.  Operands of 11 bits, 2^-12 of rounding, as long as that does not grow by
    more than it does in the usual iteration of five steps, 88 times; where it does, 22 bits.  Bounds as above, and for up to five usual steps the 1e-2 that are documented (9.5e-3 is the worst
    of ones of 1060 shapes, 7.7e-3 of 8128 identities, by the same roundings in 64 bits)."""
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(steps)
    g = alike(kind, gen).to(DTYPES[dtype])
    p, m = torch.zeros_like(g), torch.zeros(g.shape, device=DEV)
    trl_amd.muon_step_([p], [g], [m], lr=1.0, weight_decay=0.0, momentum=0.0, nesterov=False, ns_steps=steps, ns_coefficients=coefficients)
    want = -math.sqrt(max(1.0, g.shape[0] / g.shape[1])) * exact(g, steps=steps, coefficients=coefficients)
    usual, here = growth(5, (A, B, C)), growth(steps, coefficients)
    off = 12 * here * (2.0**-12 if here <= usual else 2.0**-22)
    most = 1e-2 if steps <= 5 and coefficients[0] == A else 1.0
    assert distance(p, want) <= (min(off, most) + half_step(p.dtype)) * float(want.norm()), distance(p, want) / float(want.norm())


@pytest.mark.parametrize("size", [1e-30, 1e-18, 1e-11, 1e-9, 1.0, 1e18])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_narrow_matrices_of_any_size(dtype, size):
    """64 rows or fewer, in 64 bits, however far the norm is under eps: fp32's rounding of the result, and half a step.  (Zeros are not near.)"""
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(3)
    for shape in ((50, 60), (700, 13)):
        u = (torch.randn(shape, generator=gen, device=DEV) * size).to(DTYPES[dtype])
        got, want = trl_amd.orthogonalize(u), exact(u)
        assert distance(got, want) <= (2.0**-22 + half_step(got.dtype)) * float(want.norm()), distance(got, want) / float(want.norm())


@pytest.mark.parametrize("size", [1e-16, 1e-14, 1e-12, 1e-11, 1e-10, 1.0, 1e18])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_wide_matrices_of_any_size(dtype, size):
    """Of more rows X is a multiple of 2^-38 (fp16's least number, in X's units of 2^-14): half of that is lost at the start and in each step but the last, and grows by
    3.4445 a step, 485 in all: 485 (1 + 1/3.4445 + ...) 2^-39 < 700 2^-39 in each entry.  The largest sizes have 22 bits (11 in a step) as elsewhere."""
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(4)
    for shape in ((300, 270), (70, 900)):
        u = (torch.randn(shape, generator=gen, device=DEV) * size).to(DTYPES[dtype])
        want = exact(u)
        grain = 700 * 2.0**-39 * math.sqrt(u.numel())
        got = trl_amd.orthogonalize(u)
        assert distance(got, want) <= (12 * growth(5, (A, B, C)) * 2.0**-22 + half_step(got.dtype)) * float(want.norm()) + grain
        p, m = torch.zeros_like(u), torch.zeros(shape, device=DEV)
        trl_amd.muon_step_([p], [u], [m], lr=1.0, weight_decay=0.0, momentum=0.0, nesterov=False)
        stretch = math.sqrt(max(1.0, shape[0] / shape[1]))
        # (a norm under eps shows the small singular values: those are the term a X, of 22 bits but for the last step's 11)
        bits = 12 * growth(5, (A, B, C)) * 2.0**-22 if got.dtype == torch.float32 else 1e-2
        assert distance(p, -stretch * want) <= stretch * ((bits + half_step(p.dtype)) * float(want.norm()) + grain)


def test_a_resumed_run_steps_weights_in_another_order():
    """A convolution's weight with its channels last, which AdamW steps: a run that is taken up is the run that was not."""
    import copy

    import trl_amd

    def made():
        torch.manual_seed(2)
        model = torch.nn.Sequential(torch.nn.Conv2d(3, 8, 4), torch.nn.Flatten(), torch.nn.Linear(8, 16)).to(DEV, memory_format=torch.channels_last)
        assert not model[0].weight.is_contiguous()
        return model, trl_amd.Muon(trl_amd.muon_param_groups(model), lr=0.01)

    def step(model, opt, seed):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        x = torch.randn((6, 3, 4, 4), generator=gen, device=DEV).contiguous(memory_format=torch.channels_last)
        opt.zero_grad()
        model(x).square().sum().backward()
        for p in model.parameters():  # (the library's gradients are no matter here)
            p.grad = torch.randn(p.shape, generator=gen, device=DEV).contiguous(memory_format=torch.channels_last if p.dim() == 4 else torch.contiguous_format)
        opt.step()

    whole, opt = made()
    for seed in range(4):
        step(whole, opt, seed)
        if seed == 1:
            saved = copy.deepcopy((whole.state_dict(), opt.state_dict()))
    other, again = made()
    other.load_state_dict(saved[0])
    again.load_state_dict(saved[1])
    for seed in range(2, 4):
        step(other, again, seed)
    assert all(torch.equal(p, q) for p, q in zip(whole.parameters(), other.parameters()))


def test_the_optimizers_step_in_a_graph():
    """Both kinds of groups, a learning rate on the GPU and one that is a number, replayed on new gradients with eager work between."""
    import trl_amd

    def made():
        torch.manual_seed(3)
        w = [torch.nn.Parameter(torch.randn(s, device=DEV).to(t) * 0.05) for s, t in (((90, 200), torch.bfloat16), ((16, 300), torch.float32), ((300, 70), torch.float32))]
        rest = [torch.nn.Parameter(torch.randn(s, device=DEV)) for s in ((200,), (97, 40))]
        lr = torch.tensor(0.01, device=DEV)
        return w + rest, lr, trl_amd.Muon([dict(params=w[:2], lr=lr), dict(params=w[2:], ns_steps=3), dict(params=rest, adamw=True)], lr=0.02)

    def fill(params, seed):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        for p in params:
            g = (torch.randn(p.shape, generator=gen, device=DEV) * 1e-2).to(p.dtype)
            p.grad = g if p.grad is None else p.grad.copy_(g)

    (params, lr, opt), (twins, their_lr, eager) = made(), made()
    stream = torch.cuda.Stream()
    fill(params, 0)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        opt.step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    fill(twins, 0)
    eager.step()
    for seed in range(1, 5):
        fill(params, seed)
        fill(twins, seed)
        lr.fill_(0.01 / seed)
        their_lr.fill_(0.01 / seed)
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(params, twins)), seed
        assert all(torch.equal(x, y) for p, q in zip(params, twins) for x, y in zip(opt.state[p].values(), eager.state[q].values())), seed


def test_calls_on_two_streams_at_once():
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(5)
    each = [torch.randn(s, generator=gen, device=DEV).to(t) for s, t in (((300, 500), torch.float32), ((700, 400), torch.bfloat16), ((12, 5000), torch.float32))]
    ids = torch.randint(0, 900, (9000,), generator=gen, device=DEV)
    g = torch.randn((9000, 130), generator=gen, device=DEV)
    want = trl_amd.orthogonalize(each), trl_amd.ops.embedding_bwd(g, ids, 900, 1.0, -1)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                results.append((trl_amd.orthogonalize(each), trl_amd.ops.embedding_bwd(g, ids, 900, 1.0, -1)))
    torch.cuda.synchronize()
    for xs, grad in results:
        assert all(torch.equal(x, y) for x, y in zip(xs, want[0])) and torch.equal(grad, want[1])


def test_a_patched_scaled_embedding_in_a_graph():
    """Its tensor of a scale has been read when the patch was made: no wait for the GPU in the capture."""
    import trl_amd
    from transformers.models.gemma3.modeling_gemma3 import Gemma3TextScaledWordEmbedding

    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.embed = Gemma3TextScaledWordEmbedding(97, 72, 4, embed_scale=1152**0.5)

        def get_input_embeddings(self):
            return self.embed

    model = Model().to(DEV, torch.bfloat16)
    trl_amd.patch_embedding(model)
    ids = torch.zeros((3, 50), dtype=torch.int64, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph), torch.no_grad():
        rows = model.embed(ids)
    gen = torch.Generator(device=DEV).manual_seed(1)
    for _ in range(4):
        ids.copy_(torch.randint(0, 97, ids.shape, generator=gen, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(rows, Gemma3TextScaledWordEmbedding.forward(model.embed, ids))
