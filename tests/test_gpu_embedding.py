"""Embedding lookup and its gradient (`embedding`, `embedding_grad_`, `patch_embedding`) against their definition in 64 bits.

Tolerances.  Forward: one product in fp32 (2^-24) and one rounding, half a step of the type (nothing at all with a scale of 1).
Gradient: a sum of k rows in fp32 is off by k 2^-24 of the sum of their sizes at most, the product with the scale (or, added to a value that is
there, the one rounding of the sum of both) by 2^-24 of the result, and the rounding by half a step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
WIDTHS = [1, 7, 8, 64, 1150, 2049, 4096]


def half_step(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def tiny(dtype):
    return {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134, torch.float32: 2.0**-150}[dtype]


def table(vocab, width, dtype, gen, offset=0, gap=0):
    """[vocab, width] at any alignment, with a gap between the rows."""
    store = torch.randn(offset + vocab * (width + gap), generator=gen, device=DEV).to(dtype)
    return store[offset:].view(vocab, width + gap)[:, :width]


def check_rows(got, weight, ids, scale):
    want = weight.double()[ids.long()] * scale
    assert got.shape == want.shape and got.dtype == weight.dtype
    if scale == 1.0:
        assert torch.equal(got.double(), want)
    else:
        assert bool(((got.double() - want).abs() <= (half_step(got.dtype) + 2.0**-23) * want.abs() + tiny(got.dtype)).all())


def sums64(g, ids, vocab, scale, padding, width):
    """(sums, sums of sizes, counts) of the tokens' rows, on the host: on the GPU the additions to one row wait for each other, 40 us each."""
    ids, g = ids.reshape(-1).long().cpu(), g.reshape(-1, width).double().cpu()
    kept = (ids >= 0) & (ids < vocab)
    if padding is not None:
        kept &= ids != padding
    ids, g = ids[kept], g[kept]
    zero = torch.zeros((vocab, width), dtype=torch.float64)
    count = torch.bincount(ids, minlength=vocab).double()
    return (zero.index_add(0, ids, g) * scale).to(DEV), (zero.index_add(0, ids, g.abs()) * abs(scale)).to(DEV), count.to(DEV)


def check_gradient(got, g, ids, scale, padding, was=None):
    vocab, width = got.shape
    total, sizes, count = sums64(g, ids, vocab, scale, padding, width)
    want = total if was is None else total + was.double()
    bound = (count[:, None] + 2) * 2.0**-24 * sizes + (half_step(got.dtype) + 2.0**-23) * want.abs() + tiny(got.dtype)
    off = (got.double() - want).abs()
    untouched = count == 0
    assert bool((off <= bound * 1.0001)[~untouched].all()), float((off - bound).max())
    if was is None:
        assert not got[untouched].any()
    else:
        assert torch.equal(got[untouched].nan_to_num(7.0), was[untouched].nan_to_num(7.0))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("width", WIDTHS)
def test_rows(dtype, width):
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(width)
    for shape, id_type, offset, gap, scale in [((), torch.int64, 0, 0, 1.0), ((0,), torch.int64, 0, 0, 2.0), ((1,), torch.int32, 1, 0, 1.0),
                                               ((3, 5), torch.int64, 0, 8, 0.3), ((2, 3, 129), torch.int32, 3, 5, -45.25)]:
        weight = table(211, width, DTYPES[dtype], gen, offset, gap)
        ids = torch.randint(0, 211, shape, generator=gen, device=DEV).to(id_type)
        check_rows(trl_amd.embedding(ids, weight, scale=scale), weight, ids, scale)
    ids = torch.randint(0, 211, (40, 6), generator=gen, device=DEV)
    check_rows(trl_amd.embedding(ids.t()[::2], weight, scale=0.5), weight, ids.t()[::2], 0.5)  # ids and a table in another order
    check_rows(trl_amd.embedding(ids, weight.t().contiguous().t(), scale=0.5), weight, ids, 0.5)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("tokens", [0, 1, 2, 63, 64, 65, 1000, 2047, 2049, 4097, 8192, 8193, 20000])
def test_gradient(dtype, tokens):
    import trl_amd

    t = DTYPES[dtype]
    gen = torch.Generator(device=DEV).manual_seed(tokens)
    for vocab, width, padding in [(1, 7, None), (97, 64, 96), (50257, 40, -1), (262144, 9, None)]:
        ids = torch.randint(0, vocab, (tokens,), generator=gen, device=DEV)
        if vocab == 97:
            ids[: tokens // 2] = 96  # half of them padding
            ids[tokens // 2 : tokens * 3 // 4] = 5  # and one token very often
        g = torch.randn((tokens, width), generator=gen, device=DEV).to(t)
        pad = None if padding is None else padding % vocab
        weight = table(vocab, width, t, gen).requires_grad_(True)
        rows = trl_amd.embedding(ids, weight, scale=1.7, padding_idx=padding)
        (grad,) = torch.autograd.grad(rows, weight, g)
        assert grad.dtype == t and grad.is_contiguous()
        check_gradient(grad, g, ids, 1.7, pad)
        again = torch.autograd.grad(trl_amd.embedding(ids, weight, scale=1.7, padding_idx=padding), weight, g)[0]
        assert torch.equal(grad, again)


@pytest.mark.parametrize("tokens,vocab", [(1024, 300), (1025, 300), (8191, 1 << 20), (8193, (1 << 20) - 1), (32768, 1 << 18), (32768, (1 << 20) - 1),
                                          (32769, 1000), (40000, 3), (70000, 1 << 21), (5000, 1 << 21), (16384, (1 << 18) - 1), (16384, 1 << 18),
                                          (16385, 1000), (8192, (1 << 19) - 1), (8192, 1 << 19), (1055, 1)])
def test_every_way_of_ordering(tokens, vocab):
    """Every way the tokens are brought into order, with ids all over the table, rare ones and very common ones."""
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(vocab % 1000)
    width = 11
    ids = ((vocab - 1.0) ** torch.rand((tokens,), generator=gen, device=DEV, dtype=torch.float64)).long().clamp(0, vocab - 1)
    ids[::3] = torch.randint(0, vocab, ids[::3].shape, generator=gen, device=DEV)
    ids[-1], ids[1] = vocab - 1, 0
    g = torch.randn((tokens, width), generator=gen, device=DEV)
    grad = trl_amd.ops.embedding_bwd(g, ids, vocab, 0.5, 1)
    check_gradient(grad, g, ids, 0.5, 1)
    held = torch.randn((vocab, width), generator=gen, device=DEV)
    was = held.clone()
    check_gradient(trl_amd.embedding_grad_(held, g, ids.int(), scale=0.5), g, ids, 0.5, None, was)


@pytest.mark.parametrize("tokens", [5000, 9001, 40000, 140001, (1 << 21) + 5])
def test_most_tokens_are_one(tokens):
    """Image placeholders, for instance.  The sums of 16 places, of 16 such sums and so on, with runs that begin and end anywhere in them."""
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(tokens)
    vocab, width = 4000, 24
    for share in (0.6, 1.0):
        ids = torch.randint(0, vocab, (tokens,), generator=gen, device=DEV)
        often = torch.rand((tokens,), generator=gen, device=DEV)
        ids[often < share] = 1777
        ids[(often < share) & (often > 0.8 * share)] = 1778
        g = torch.randn((tokens, width), generator=gen, device=DEV).bfloat16()
        check_gradient(trl_amd.ops.embedding_bwd(g, ids, vocab, 1.0, -1), g, ids, 1.0, None)


@pytest.mark.parametrize("dtype,into", [("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32"), ("fp32", "fp32")])
@pytest.mark.parametrize("tokens", [1, 300, 3000, 9000])
def test_added_gradient(dtype, into, tokens):
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(tokens + 1)
    for width, offset, gap, id_type in [(1150, 0, 0, torch.int64), (37, 3, 6, torch.int32), (2056, 0, 8, torch.int64)]:
        vocab = 701
        was = table(vocab, width, DTYPES[into], gen, offset, gap).clone(memory_format=torch.preserve_format)
        was[700] = math.nan  # of a token that does not occur
        buffer = torch.full((vocab, width + gap), 3.0, dtype=DTYPES[into], device=DEV)
        held = buffer[:, :width]
        held.copy_(was)
        ids = torch.randint(0, 700, (tokens,), generator=gen, device=DEV).to(id_type)
        g = torch.randn((tokens, width + 3), generator=gen, device=DEV).to(DTYPES[dtype])[:, :width]  # rows apart
        assert trl_amd.embedding_grad_(held, g, ids, scale=0.25, padding_idx=11) is held
        check_gradient(held, g, ids, 0.25, 11, was)
        if gap:
            assert bool((buffer[:, width:] == 3.0).all())


def test_differences():
    """Small whole numbers: every product and sum is exact, and so is the difference that one entry of the table makes."""
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(1)
    weight = torch.randint(-4, 5, (13, 6), generator=gen, device=DEV).float().requires_grad_(True)
    ids = torch.randint(0, 13, (5, 9), generator=gen, device=DEV)
    u = torch.randint(-4, 5, (5, 9, 6), generator=gen, device=DEV).float()
    loss = lambda w: (trl_amd.embedding(ids, w, scale=2.0) * u).sum()  # noqa: E731
    (grad,) = torch.autograd.grad(loss(weight), weight)
    with torch.no_grad():
        for v in range(13):
            for k in range(6):
                moved = weight.detach().clone()
                moved[v, k] += 1.0
                assert float(loss(moved) - loss(weight)) == float(grad[v, k])


def test_ids_outside_the_table():
    import trl_amd

    trl_amd.check_device_errors()
    weight = torch.randn((50, 20), device=DEV, requires_grad=True)
    for bad in (-1, 50, 1 << 40, -(1 << 40)):
        ids = torch.tensor([3, bad, 4, 3], device=DEV)
        rows = trl_amd.embedding(ids, weight, scale=2.0)
        assert bool(rows[1].isnan().all()) and torch.equal(rows[[0, 2, 3]], 2.0 * weight[[3, 4, 3]])
        with pytest.raises(IndexError):
            trl_amd.check_device_errors()
        (grad,) = torch.autograd.grad(rows, weight, torch.ones_like(rows))
        with pytest.raises(IndexError):
            trl_amd.check_device_errors()
        assert float(grad[3, 0]) == 4.0 and float(grad[4, 0]) == 2.0 and float(grad.sum()) == 120.0
    trl_amd.check_device_errors()


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_large_outputs(dtype):
    """Outputs that go past the caches, with cut rows."""
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(8)
    weight = table(5000, 2049, DTYPES[dtype], gen)
    ids = torch.randint(0, 5000, (70000 if dtype != "fp32" else 35000,), generator=gen, device=DEV)
    rows = trl_amd.embedding(ids, weight, scale=0.5)
    for part in (slice(0, 100), slice(17000, 17100), slice(-100, None)):
        check_rows(rows[part], weight, ids[part], 0.5)
    assert torch.equal(rows, trl_amd.embedding(ids.flip(0), weight, scale=0.5).flip(0))


def test_infinities_and_nan_stay_in_their_rows():
    import trl_amd

    weight = torch.randn((9, 33), device=DEV, dtype=torch.bfloat16)
    weight[2], weight[3, 5] = math.inf, math.nan
    rows = trl_amd.embedding(torch.tensor([2, 3, 4], device=DEV), weight, scale=0.5)
    assert bool(rows[0].isinf().all()) and int(rows[1].isnan().sum()) == 1 and bool(rows[2].isfinite().all())
    g = torch.randn((4, 33), device=DEV)
    g[1, 7] = math.nan
    g[3] = math.inf
    held = torch.zeros((9, 33), device=DEV)
    trl_amd.embedding_grad_(held, g, torch.tensor([5, 6, 5, 0], device=DEV), padding_idx=0)  # (the infinite one is padding)
    assert int(held.isnan().sum()) == 1 and bool(held[6, 7].isnan()) and not held[0].any() and not held.isinf().any()


def test_offsets_past_32_bits():
    import trl_amd

    vocab, width = 262144, 9000  # 2.36e9 entries
    weight = torch.empty((vocab, width), dtype=torch.bfloat16, device=DEV)
    some = torch.tensor([0, 1, 238609, 238610, 262143], device=DEV)
    weight[some] = torch.randn((5, width), device=DEV).bfloat16()
    ids = some.repeat(3)
    assert torch.equal(trl_amd.embedding(ids, weight), weight[ids])
    g = torch.randn((15, width), device=DEV).bfloat16()
    grad = torch.autograd.grad(trl_amd.embedding(ids, weight.requires_grad_(True)), weight, g)[0]
    want = g.double().view(3, 5, width).sum(0)
    assert bool(((grad[some].double() - want).abs() <= 2.0**-7 * want.abs() + 2.0**-20).all())
    grad[some] = 0
    assert not grad.any()
    del grad, weight
    # and of the tokens: 70000 rows of 32768 entries
    g = torch.zeros((70000, 32768), dtype=torch.bfloat16, device=DEV)
    g[[0, 65535, 65536, 69999]] = 1.0
    ids = torch.arange(70000, device=DEV) % 7
    held = torch.zeros((7, 32768), device=DEV)
    trl_amd.embedding_grad_(held, g, ids)
    want = torch.zeros(7, device=DEV)
    for i in (0, 65535, 65536, 69999):
        want[i % 7] += 1
    assert torch.equal(held, want[:, None].expand(7, 32768))


def test_other_streams_and_inference_mode():
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(4)
    weight = table(300, 520, torch.bfloat16, gen).requires_grad_(True)
    ids = torch.randint(0, 300, (2, 500), generator=gen, device=DEV)
    g = torch.randn((2, 500, 520), generator=gen, device=DEV).bfloat16()
    want = torch.autograd.grad(trl_amd.embedding(ids, weight, scale=3.0), weight, g)[0]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = torch.autograd.grad(trl_amd.embedding(ids, weight, scale=3.0), weight, g)[0]
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)
    with torch.inference_mode():
        rows = trl_amd.embedding(ids, weight, scale=3.0)
        assert not rows.requires_grad
        trl_amd.embedding_grad_(torch.zeros((300, 520), device=DEV), g, ids)


@pytest.mark.parametrize("tokens", [100, 4000, 12000])
def test_graph_capture(tokens):
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(9)
    weight = table(400, 264, torch.float32, gen).requires_grad_(True)
    ids = torch.randint(0, 400, (tokens,), generator=gen, device=DEV)
    g = torch.randn((tokens, 264), generator=gen, device=DEV)
    held = torch.zeros((400, 264), device=DEV)

    def step():
        rows = trl_amd.embedding(ids, weight, scale=0.5, padding_idx=3)
        grad = torch.autograd.grad(rows, weight, g)[0]
        trl_amd.embedding_grad_(held, g, ids)
        return rows, grad

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows, grad = step()
    for seed in range(4):
        ids.copy_(torch.randint(0, 400, (tokens,), generator=gen, device=DEV))
        g.normal_(generator=gen)
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = held.clone()
        assert torch.equal(rows, weight[ids] * 0.5)
        check_gradient(grad, g, ids, 0.5, 3)
        held.zero_()
        want = trl_amd.embedding_grad_(torch.zeros_like(held), g, ids)
        assert torch.equal(got, want)


def test_what_has_no_derivative_raises():
    import trl_amd

    weight = torch.randn((20, 16), device=DEV, requires_grad=True)
    ids = torch.arange(10, device=DEV)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda w: trl_amd.embedding(ids, w), (weight.detach(),), (torch.ones_like(weight),))
    (grad,) = torch.autograd.grad(trl_amd.embedding(ids, weight).square().sum(), weight, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_gradients_of_broadcast_and_summed_rows():
    import trl_amd

    gen = torch.Generator(device=DEV).manual_seed(2)
    weight = table(60, 24, torch.float32, gen).requires_grad_(True)
    ids = torch.randint(0, 60, (3, 7), generator=gen, device=DEV)
    (grad,) = torch.autograd.grad(trl_amd.embedding(ids, weight, scale=0.5).sum(), weight)  # one number for all entries
    assert torch.equal(grad, 0.5 * torch.bincount(ids.flatten(), minlength=60).float()[:, None].expand(60, 24))
    u = torch.randn((7, 3, 24), generator=gen, device=DEV).transpose(0, 1)
    (grad,) = torch.autograd.grad(trl_amd.embedding(ids, weight), weight, u)
    check_gradient(grad, u, ids, 1.0, None)


def test_refused_memory_and_types():
    import trl_amd

    held, ids = torch.zeros((30, 8), device=DEV), torch.arange(4, device=DEV)
    for g, error in ((held[:4], ValueError), (torch.zeros((4, 7), device=DEV), ValueError), (torch.zeros((5, 8), device=DEV), ValueError),
                     (torch.zeros((4, 8), device=DEV, dtype=torch.float64), TypeError), (torch.zeros((4, 8)), RuntimeError)):
        with pytest.raises(error):
            trl_amd.embedding_grad_(held, g, ids)
    with pytest.raises(TypeError):
        trl_amd.embedding_grad_(held.half(), torch.zeros((4, 8), device=DEV), ids)
    with pytest.raises(ValueError):
        trl_amd.embedding_grad_(held.t(), torch.zeros((4, 30), device=DEV), ids)
    for bad, error in ((ids.float(), TypeError), (ids.short(), TypeError), (ids.cpu(), RuntimeError)):
        with pytest.raises(error):
            trl_amd.embedding(bad, held)
    with pytest.raises(TypeError):
        trl_amd.embedding(ids, held.double())
    with pytest.raises(ValueError):
        trl_amd.embedding(ids, held[0])


class Tied(torch.nn.Module):
    def __init__(self, embed):
        super().__init__()
        self.embed = embed

    def get_input_embeddings(self):
        return self.embed

    def forward(self, ids):
        return self.embed(ids)


def test_patched_modules():
    import trl_amd
    from transformers.models.gemma3.modeling_gemma3 import Gemma3TextScaledWordEmbedding

    torch.manual_seed(0)
    ids = torch.randint(0, 97, (3, 50), device=DEV)
    for make in (lambda: torch.nn.Embedding(97, 72, padding_idx=4), lambda: torch.nn.Embedding(97, 72),
                 lambda: Gemma3TextScaledWordEmbedding(97, 72, 4, embed_scale=72**0.5)):
        for dtype in (torch.float32, torch.bfloat16):
            model = Tied(make()).to(DEV, dtype)
            want = model(ids)
            g = torch.randint(-8, 9, want.shape, device=DEV).to(dtype)
            grad = torch.autograd.grad(want, model.embed.weight, g)[0]
            trl_amd.patch_embedding(model)
            got = model(ids)
            assert torch.equal(got, want)
            mine = torch.autograd.grad(got, model.embed.weight, g)[0]
            # (torch adds bf16 gradients in fp32 and rounds the scaled rows before; both sides are near)
            torch.testing.assert_close(mine, grad, rtol=2e-2 if dtype == torch.bfloat16 else 1e-5, atol=0.25 if dtype == torch.bfloat16 else 1e-3)
            if type(model.embed) is torch.nn.Embedding and dtype == torch.float32:
                assert torch.equal(mine, grad)  # whole numbers: exact


def test_patched_modules_after_a_cast_and_compiled():
    """A model that is cast after the patch, and one that is compiled, have the module's own rows, and gradients."""
    import trl_amd
    from transformers.models.bart.modeling_bart import BartScaledWordEmbedding
    from transformers.models.gemma3.modeling_gemma3 import Gemma3TextScaledWordEmbedding

    torch.manual_seed(0)
    ids = torch.randint(0, 97, (3, 50), device=DEV)
    for make in (lambda: torch.nn.Embedding(97, 72, padding_idx=4), lambda: Gemma3TextScaledWordEmbedding(97, 72, 4, embed_scale=1152**0.5),
                 lambda: BartScaledWordEmbedding(97, 72, 4, embed_scale=1152**0.5)):
        model = Tied(make())
        trl_amd.patch_embedding(model)
        for dtype in (torch.float32, torch.bfloat16):
            model.to(DEV, dtype)
            own = type(model.embed).forward
            torch._dynamo.reset()
            for call in (model, torch.compile(model, backend="aot_eager", fullgraph=True)):
                want, got = own(model.embed, ids), call(ids)
                assert torch.equal(got, want)
                g = torch.randint(-8, 9, want.shape, device=DEV).to(dtype)
                grads = [torch.autograd.grad(x, model.embed.weight, g)[0] for x in (want, got)]
                # whole numbers times one factor: exact sums, but for the rounding of each product (half a step each, of 3 and more of one token)
                step = 0.0 if type(model.embed) is torch.nn.Embedding else torch.finfo(dtype).eps
                size = torch.autograd.grad(own(model.embed, ids), model.embed.weight, g.abs())[0].double()
                assert bool(((grads[1].double() - grads[0].double()).abs() <= 2 * step * size).all())
