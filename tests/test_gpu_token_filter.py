"""Tokens drawn from, and scored under, a filtered distribution (`sample_tokens`, `filtered_logps`) against their definition in
64 bits on the host: a row's tokens sorted by (logit descending, index ascending), each filter a prefix of that order.

Tolerances.  Ids are equal.  A log-prob is computed in 64 bits from weights in units of 2^-fix, 62 - fix the number of the
vocabulary's bits, and rounded to fp32 once: 2^-24 of its size, V 2^-(fix+1) for the weights and 1e-11 for exp2 and log2.
A gradient entry is g / T * (1[v = id] - p) with p = 2^t in fp32, t off by at most 3 * 64 * 2^-24 where p counts, so p by
ln 2 * 1.2e-5 < 1e-5 of itself, and half a step of the output's type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def row_support(x, T, k, p, q):
    """Kept tokens of one row of 64-bit logits, in index order, and their weights (the largest 1)."""
    if T == 0:
        T, k = 1.0, 1
    order = torch.argsort(-x, stable=True)
    order = order[x[order] > -math.inf]
    if k > 0:
        order = order[:k]
    w = ((x[order] - x[order[0]]) / T).exp()
    if p < 1:
        before = w.cumsum(0) - w
        n = max(1, int((before < p * w.sum()).sum()))
        order, w = order[:n], w[:n]
    keep = w >= q
    order, w = order[keep], w[keep]
    at = order.argsort()
    return order[at], w[at]


def _setting(value, i):
    return value.reshape(-1)[i].item() if torch.is_tensor(value) else value


def expected(logits, s, uniforms=None, ids=None):
    """(ids, logps) drawn, or logps of `ids` and the probabilities [rows, V] of the kept tokens."""
    x = logits.detach().double().cpu().reshape(-1, logits.shape[-1])
    out_ids, out_logps, probs = [], [], torch.zeros_like(x) if ids is not None else None
    for r in range(x.shape[0]):
        tokens, w = row_support(x[r], *(_setting(s[n], r) for n in ("temperature", "top_k", "top_p", "min_p")))
        c = w.cumsum(0)
        if ids is None:
            at = min(int((c <= uniforms.double().cpu().reshape(-1)[r] * c[-1]).sum()), len(c) - 1)
            out_ids.append(int(tokens[at]))
            out_logps.append(math.log(float(w[at] / c[-1])) if float(w[at]) > 0 else -math.inf)
        else:
            probs[r, tokens] = w / c[-1]
            t = int(ids.reshape(-1)[r])
            hit = (tokens == t).nonzero()
            out_logps.append(math.log(float(w[hit[0, 0]] / c[-1])) if len(hit) else -math.inf)
    lp = torch.tensor(out_logps, dtype=torch.float64)
    return (torch.tensor(out_ids), lp) if ids is None else (lp, probs)


def close(got, want, V):
    got = got.double().cpu().reshape(-1)
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), (got, want)
    f = torch.isfinite(want)
    bound = 2.0**-24 * want[f].abs() + V * 2.0 ** -(63 - V.bit_length()) + 1e-11
    off = (got[f] - want[f]).abs()
    assert bool((off <= bound).all()), (off.max(), got[f][off > bound], want[f][off > bound])


def settings(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    return dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)


FILTERS = [
    settings(), settings(0.7), settings(0.7, 50), settings(1.0, 1), settings(1.3, 7), settings(1.0, 0, 0.9), settings(0.6, 0, 0.5),
    settings(0.9, 20, 0.8), settings(1.0, 0, 1.0, 0.05), settings(1.0, 0, 0.95, 0.02), settings(0.8, 40, 0.95, 0.1), settings(0.0),
    settings(1.0, 64, 1.0, 0.3), settings(1.0, 0, 1e-6), settings(1.0, 10**6, 1.0, 1.0),
]
VOCABS = [1, 2, 63, 64, 65, 1000, 2047, 2048, 2049, 4100, 32001]


def make_logits(rows, V, dtype, seed, slope=1.7):
    g = torch.Generator().manual_seed(seed)
    x = torch.empty(rows, V).exponential_(generator=g) * slope - 3.0
    return x.to(DTYPES[dtype]), torch.rand(rows, generator=g)


def draw(logits, u, s, **kw):
    import trl_amd

    s = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in s.items()}
    ids, lp = trl_amd.sample_tokens(logits.to(DEV), u.to(DEV), **s, **kw)
    trl_amd.check_device_errors()
    return ids.cpu(), lp


def check_draw(logits, u, s):
    ids, lp = draw(logits, u, s)
    want_ids, want = expected(logits, s, uniforms=u)
    assert torch.equal(ids.reshape(-1), want_ids), (s, ids.reshape(-1)[ids.reshape(-1) != want_ids], want_ids[ids.reshape(-1) != want_ids])
    close(lp, want, logits.shape[-1])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", VOCABS)
def test_drawn_tokens(V, dtype):
    for i, s in enumerate(FILTERS):
        logits, u = make_logits(7, V, dtype, 100 * i + V)
        check_draw(logits, u, s)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_ties_go_by_index(dtype):
    """Whole logits: every border lies inside a class of equal tokens, of which the first are kept."""
    g = torch.Generator().manual_seed(5)
    for V in (8, 200, 5000):
        for hi in (1, 3, 30):
            logits = torch.randint(0, hi, (9, V), generator=g).to(DTYPES[dtype])
            u = torch.rand(9, generator=g)
            for s in (settings(1.0, 5), settings(1.0, V // 2), settings(1.0, 0, 0.5), settings(0.7, 0, 0.37), settings(1.0, V // 3, 0.5),
                      settings(1.0, 0, 1.0, 0.1), settings(1.0, 0, 0.6, 0.3), settings(0.0), settings()):
                check_draw(logits, u, s)


def test_signed_zeros_are_equal():
    logits = torch.tensor([[-0.0, 0.0, -0.0, 0.0, -1.0]]).repeat(4, 1)
    u = torch.tensor([0.0, 0.3, 0.6, 0.99])
    for dtype in DTYPES.values():
        for s in (settings(1.0, 2), settings(1.0, 3), settings(1.0, 0, 0.4), settings(0.0)):
            check_draw(logits.to(dtype), u, s)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_masked_logits(dtype):
    """-inf and the type's lowest value, on the leading, trailing and most tokens; one token left."""
    V, t = 5000, DTYPES[dtype]
    g = torch.Generator().manual_seed(11)
    base, u = make_logits(8, V, dtype, 12)
    u[0], u[1] = 0.0, 1.0 - 2.0**-24
    for value in (-math.inf, torch.finfo(t).min):
        rows = []
        for r in range(8):
            x = base[r].clone()
            if r % 4 == 0:
                x[: 3000] = value
            elif r % 4 == 1:
                x[2500:] = value
            elif r % 4 == 2:
                x[torch.rand(V, generator=g) < 0.995] = value
            else:
                x[:] = value
                x[4321] = 1.0
            rows.append(x)
        logits = torch.stack(rows)
        for s in FILTERS:
            if value != -math.inf and s["temperature"] < 1 and s["top_k"] == 50:
                continue  # (more tokens than are left: the same as without)
            check_draw(logits, u, s)
    for s in FILTERS:  # nothing but the lowest value: all equal
        check_draw(torch.full((3, 70), torch.finfo(t).min, dtype=t), torch.tensor([0.0, 0.4, 0.999]), s)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_flat_rows_have_more_candidates_than_are_held(dtype):
    g = torch.Generator().manual_seed(3)
    logits = (0.3 * torch.randn(4, 50001, generator=g)).to(DTYPES[dtype])
    logits[3] = 0.25  # all equal
    u = torch.rand(4, generator=g)
    for s in (settings(1.0, 0, 0.9), settings(0.5, 5000), settings(1.0, 20000, 0.6), settings(1.0, 0, 1.0, 0.5), settings(),
              settings(1.0, 30000, 0.99, 0.4), settings(1.0, 3)):
        check_draw(logits, u, s)


def test_large_vocabulary():
    logits, u = make_logits(3, 300007, "bf16", 21, slope=1.3)
    for s in (settings(), settings(1.0, 50), settings(1.0, 0, 0.95), settings(0.8, 100, 0.9, 0.01)):
        check_draw(logits, u, s)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("slope", [0.7, 1.0, 1.3, 2.0])
def test_every_number_of_candidates(slope, dtype):
    """Nuclei and top-k of a few tokens to most of the vocabulary: rows whose candidates are compared in pairs, binned in LDS, or found
    by passes over the row, drawn from and scored."""
    import trl_amd

    logits, u = make_logits(4, 60013, dtype, int(10 * slope), slope)
    logits[3, ::3] = -math.inf
    for s in (settings(1.0, 127), settings(1.0, 128), settings(1.0, 129), settings(0.9, 700), settings(1.0, 3000), settings(1.0, 5000),
              settings(1.0, 400, 0.9), settings(1.0, 0, 0.3), settings(1.0, 0, 0.7), settings(1.0, 0, 0.9), settings(1.0, 0, 0.99),
              settings(1.0, 0, 0.9999), settings(1.0, 0, 1.0, 1e-3), settings(1.0, 0, 1.0, 1e-5), settings(1.0, 0, 0.99, 1e-4),
              settings(1.0, 2000, 1.0, 1e-3), settings(3.0, 0, 0.9), settings(3.0, 900)):
        check_draw(logits, u, s)
        ids, lp = trl_amd.sample_tokens(logits.to(DEV), u.to(DEV), **s)
        assert torch.equal(trl_amd.filtered_logps(logits.to(DEV), ids, **s), lp)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_long_nuclei_and_their_gradient(dtype):
    g = torch.Generator().manual_seed(17)
    logits, _ = make_logits(4, 30011, dtype, 18, 1.05)
    for s in (settings(1.0, 0, 0.9), settings(1.0, 0, 0.99, 1e-4), settings(1.0, 1500), settings(1.0, 0, 1.0, 1e-4), settings(1.0, 300, 0.95)):
        ids = torch.stack([row_support(x.double(), 1.0, s["top_k"], s["top_p"], s["min_p"])[0][-1] for x in logits])
        ids[0] = int(logits[0].argmin())
        check_score(logits, ids, s, torch.randn(4, generator=g))


def test_offsets_past_32_bits():
    """Rows that start behind 2^31 and 2^32 entries of their tensor, and a gradient of more than 2^32."""
    import trl_amd

    V, rows = 262144, 16400  # 4.3e9 entries
    if torch.cuda.mem_get_info()[0] < 24 * 2**30:
        pytest.skip("needs 24 GiB of GPU memory")
    logits = torch.zeros((rows, V), dtype=torch.bfloat16, device=DEV)
    mask = torch.zeros(rows, dtype=torch.bool, device=DEV)
    at = torch.tensor([0, 8191, 8192, 8193, 16383, 16384, 16399])
    few, u = make_logits(len(at), V, "bf16", 19)
    logits[at.to(DEV)] = few.to(DEV)
    mask[at.to(DEV)] = True
    uniforms = torch.zeros(rows, device=DEV)
    uniforms[at.to(DEV)] = u.to(DEV)
    s = settings(1.0, 30, 0.9)
    ids, lp = trl_amd.sample_tokens(logits, uniforms, **s, row_mask=mask)
    want_ids, want = expected(few, s, uniforms=u)
    assert torch.equal(ids.cpu()[at], want_ids)
    close(lp.cpu()[at], want, V)
    x = logits.requires_grad_(True)
    scored = trl_amd.filtered_logps(x, ids, **s, row_mask=mask)
    assert torch.equal(scored.detach()[at.to(DEV)], lp[at.to(DEV)])
    (grad,) = torch.autograd.grad(scored, x, torch.ones_like(scored))
    y = few.to(DEV).requires_grad_(True)
    (small,) = torch.autograd.grad(trl_amd.filtered_logps(y, want_ids.to(DEV), **s).sum(), y)
    assert torch.equal(grad[at.to(DEV)], small)
    assert int(grad.any(-1).sum()) == int(small.any(-1).sum())  # (a row that keeps one token has the gradient 1 - 1)


@pytest.mark.parametrize("temperature", [1e-4, 0.05, 30.0, 1e4])
def test_temperatures(temperature):
    logits, u = make_logits(6, 3001, "fp32", 31)
    logits[0] += 1000.0
    logits[1] -= 1e6
    for s in (settings(temperature), settings(temperature, 9), settings(temperature, 0, 0.9), settings(temperature, 0, 1.0, 0.2)):
        check_draw(logits, u, s)


def test_a_value_for_each_row():
    rows, V = 48, 4099
    for dtype in DTYPES:
        logits, u = make_logits(rows, V, dtype, 41)
        g = torch.Generator().manual_seed(42)
        pick = lambda values, t: torch.tensor(values, dtype=t)[torch.randint(0, len(values), (rows,), generator=g)]  # noqa: E731
        s = settings(pick([0.0, 0.5, 1.0, 2.0], torch.float32), pick([0, -1, 1, 30, V, 10**6], torch.int32),
                     pick([1.0, 0.9, 0.4], torch.float32), pick([0.0, 0.0, 0.1, 1.0], torch.float32))
        check_draw(logits, u, s)
        check_draw(logits, u, dict(s, temperature=0.8, top_p=1.0))
        check_draw(logits, u, dict(settings(), top_k=s["top_k"].long()))


def test_uniform_numbers_at_the_ends():
    logits, _ = make_logits(4, 3000, "bf16", 51)
    logits[:, 0] = -math.inf
    for u in (torch.zeros(4), torch.full((4,), 1.0 - 2.0**-24), torch.full((4,), 1.0 - 2.0**-53, dtype=torch.float64)):
        for s in (settings(), settings(1.0, 30), settings(1.0, 0, 0.9), settings(1.0, 0, 1.0, 0.01)):
            ids, lp = draw(logits, u, s)
            if u.dtype == torch.float32 and float(u[0]):  # (a last token of less than 2^-24 lies behind that number)
                assert torch.equal(ids, expected(logits, s, uniforms=u)[0])
                continue
            for r in range(4):
                tokens, _ = row_support(logits[r].double(), *(s[n] for n in ("temperature", "top_k", "top_p", "min_p")))
                assert int(ids[r]) == int(tokens[0] if float(u[r]) == 0.0 else tokens[-1])


def test_strides_and_alignment():
    import trl_amd

    g = torch.Generator().manual_seed(61)
    for dtype in DTYPES.values():
        store = torch.randn(6 * 5 * 1003 + 3, generator=g).mul(2).to(dtype)
        base = store[3:].view(6, 5, 1003)
        on = store.to(DEV)[3:].view(6, 5, 1003)  # (an odd element offset)
        for cut in (lambda t: t[:, -1], lambda t: t[:, 1:4], lambda t: t[::2, 2], lambda t: t[:, :, 1:900], lambda t: t[0, 0],
                    lambda t: t.transpose(0, 1), lambda t: t[:1].expand(3, 5, 1003)):
            x, y = cut(base), cut(on)
            u = torch.rand(x.shape[:-1], generator=g)
            for s in (settings(0.9), settings(1.0, 20, 0.9)):
                ids, lp = trl_amd.sample_tokens(y, u.to(DEV), **s)
                assert ids.shape == lp.shape == x.shape[:-1]
                want_ids, want = expected(x.contiguous(), s, uniforms=u)
                assert torch.equal(ids.cpu().reshape(-1), want_ids)
                close(lp, want, x.shape[-1])


def test_a_rows_token_does_not_depend_on_the_batch():
    import trl_amd

    logits, u = make_logits(300, 20011, "bf16", 71)
    x, v = logits.to(DEV), u.to(DEV)
    for s in (settings(), settings(1.0, 50, 0.9), settings(1.0, 0, 0.95)):
        ids, lp = trl_amd.sample_tokens(x, v, **s)
        for r in (0, 17, 299):
            one, lp1 = trl_amd.sample_tokens(x[r : r + 1], v[r : r + 1], **s)
            assert torch.equal(one, ids[r : r + 1]) and torch.equal(lp1, lp[r : r + 1])
        again = trl_amd.sample_tokens(x, v, **s)
        assert torch.equal(again[0], ids) and torch.equal(again[1], lp)


def test_masked_rows_are_left_alone():
    import trl_amd

    logits, u = make_logits(6, 3000, "bf16", 81)
    mask = torch.tensor([1, 0, 1, 0, 1, 1])
    logits[1] = math.nan  # (a masked row is not looked at)
    for s in (settings(), settings(1.0, 20)):
        ids, lp = draw(logits, u, s, row_mask=mask.to(DEV), pad_token_id=777)
        on = mask.bool()
        want_ids, want = expected(logits[on], s, uniforms=u[on])
        assert torch.equal(ids[on], want_ids) and bool((ids[~on] == 777).all())
        close(lp.cpu()[on], want, 3000)
        assert bool((lp.cpu()[~on] == 0).all())
        x = logits.to(DEV).requires_grad_(True)
        lp = trl_amd.filtered_logps(x, ids.clamp(max=2999).to(DEV), **s, row_mask=mask.bool().to(DEV))
        (grad,) = torch.autograd.grad(lp, x, torch.ones_like(lp))
        assert bool((lp.cpu()[~on] == 0).all()) and bool((grad.cpu()[~on] == 0).all()) and bool((grad.cpu()[on] != 0).any())
        trl_amd.check_device_errors()


def test_rows_without_a_distribution():
    import trl_amd

    for V in (10, 3000):
        for s in (settings(), settings(1.0, 5), settings(1.0, 0, 0.9), settings(0.0)):
            logits, u = make_logits(6, V, "bf16", 91)
            logits[0] = -math.inf
            logits[2, V // 2] = math.nan
            logits[3, V - 1] = math.inf
            logits[5, 0] = -math.nan
            ids, lp = trl_amd.sample_tokens(logits.to(DEV), u.to(DEV), **s)
            with pytest.raises(ValueError, match="no distribution"):
                trl_amd.check_device_errors()
            trl_amd.check_device_errors()  # (told once)
            bad = torch.tensor([0, 2, 3, 5])
            assert bool((ids.cpu()[bad] == -1).all()) and bool(lp.cpu()[bad].isnan().all())
            good = torch.tensor([1, 4])
            want_ids, want = expected(logits[good], s, uniforms=u[good])
            assert torch.equal(ids.cpu()[good], want_ids)
            close(lp.cpu()[good], want, V)
            x = logits.to(DEV).requires_grad_(True)
            lp = trl_amd.filtered_logps(x, torch.zeros(6, dtype=torch.long, device=DEV), **s)
            (grad,) = torch.autograd.grad(lp, x, torch.ones_like(lp))
            assert bool(lp.cpu()[bad].isnan().all()) and bool((grad.cpu()[bad] == 0).all())
            with pytest.raises(ValueError, match="no distribution"):
                trl_amd.check_device_errors()
    # a row's own setting that is none
    logits, u = make_logits(4, 100, "fp32", 92)
    ids, lp = trl_amd.sample_tokens(logits.to(DEV), u.to(DEV), temperature=torch.tensor([1.0, -1.0, math.nan, math.inf], device=DEV))
    assert ids[1:].tolist() == [-1, -1, -1] and int(ids[0]) >= 0
    with pytest.raises(ValueError, match="no distribution"):
        trl_amd.check_device_errors()


# ---- scoring ---------------------------------------------------------------------------------------------------------
def check_score(logits, ids, s, g):
    import trl_amd

    on = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in s.items()}
    x = logits.to(DEV).requires_grad_(True)
    lp = trl_amd.filtered_logps(x, ids.to(DEV), **on)
    want, probs = expected(logits, s, ids=ids)
    V = logits.shape[-1]
    close(lp.detach(), want, V)
    (grad,) = torch.autograd.grad(lp, x, g.to(DEV))
    assert grad.dtype == logits.dtype and grad.shape == logits.shape and grad.is_contiguous()
    trl_amd.check_device_errors()
    T = s["temperature"].double().reshape(-1) if torch.is_tensor(s["temperature"]) else torch.full((len(want),), float(s["temperature"]), dtype=torch.float64)
    T = torch.where(T == 0, 1.0, T)
    one = torch.nn.functional.one_hot(ids.reshape(-1), V).double()
    scale = (g.double().reshape(-1) / T * torch.isfinite(want))[:, None]
    exact = scale * (one - probs)
    bound = scale.abs() * (1e-5 * probs + 2.0**-22 * one) + exact.abs() * torch.finfo(logits.dtype).eps / 2 + torch.finfo(logits.dtype).tiny
    off = (grad.double().cpu().reshape(-1, V) - exact).abs()
    assert bool((off <= bound).all()), (s, (off - bound).max())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [1, 2, 64, 65, 1000, 2049, 9001])
def test_scored_tokens_and_their_gradient(V, dtype):
    for i, s in enumerate(FILTERS):
        logits, _ = make_logits(10, V, dtype, 7 * i + V)
        g = torch.Generator().manual_seed(i)
        leading = logits.float().topk(min(V, 12), dim=-1).indices
        ids = leading.gather(1, torch.randint(0, leading.shape[1], (10, 1), generator=g)).squeeze(1)
        ids[0] = int(torch.randint(0, V, (1,), generator=g))
        check_score(logits.view(2, 5, V), ids.view(2, 5), s, torch.randn(2, 5, generator=g))


def test_scored_ties_and_masks():
    g = torch.Generator().manual_seed(8)
    for dtype in DTYPES.values():
        logits = torch.randint(0, 4, (12, 700), generator=g).to(dtype)
        logits[3, 100:] = -math.inf
        logits[4, :] = torch.finfo(dtype).min
        for s in (settings(1.0, 60), settings(0.8, 0, 0.5), settings(1.0, 300, 0.7), settings(1.0, 0, 1.0, 0.2), settings(), settings(0.0)):
            ids = torch.randint(0, 700, (12,), generator=g)
            ids[3] = 50
            check_score(logits, ids, s, torch.randn(12, generator=g))


def test_scored_with_a_value_for_each_row():
    rows, V = 24, 2500
    logits, _ = make_logits(rows, V, "fp32", 141)
    g = torch.Generator().manual_seed(142)
    pick = lambda values, t: torch.tensor(values, dtype=t)[torch.randint(0, len(values), (rows,), generator=g)]  # noqa: E731
    s = settings(pick([0.0, 0.5, 1.0], torch.float32), pick([0, 1, 30], torch.int32), pick([1.0, 0.9], torch.float32),
                 pick([0.0, 0.1], torch.float32))
    check_score(logits, logits.argmax(-1), s, torch.randn(rows, generator=g))


def test_gradient_against_differences():
    """Central differences of the definition in 64 bits, with a support that does not change within the step (the border's
    distance to the next logit is looked at)."""
    import trl_amd

    logits, _ = make_logits(3, 40, "fp32", 151)
    s, h = settings(0.8, 12), 1e-4
    order = logits.double().sort(dim=-1, descending=True)
    assert float((order.values[:, 11] - order.values[:, 12]).min()) > 4 * h
    ids = order.indices[:, 3]
    x = logits.to(DEV).requires_grad_(True)
    (grad,) = torch.autograd.grad(trl_amd.filtered_logps(x, ids.to(DEV), **s).sum(), x)
    for r in range(3):
        for v in range(40):
            at = []
            for sign in (1, -1):
                y = logits.double().clone()
                y[r, v] += sign * h
                at.append(float(expected(y, s, ids=ids)[0][r]))
            # (third derivatives of a log-softmax are under 1 / T^3 = 2: h^2 / 6 * 2, and 1e-15 / h of rounding)
            assert abs(float(grad[r, v]) - (at[0] - at[1]) / (2 * h)) < 1e-8 + 1e-5 * 1.25 + 2.0**-22


def test_ids_outside_the_vocabulary():
    import trl_amd

    logits, _ = make_logits(4, 100, "fp32", 161)
    x = logits.to(DEV).requires_grad_(True)
    for s in (settings(), settings(1.0, 5)):
        lp = trl_amd.filtered_logps(x, torch.tensor([-1, 100, 2**40, int(logits[3].argmax())], device=DEV), **s)
        (grad,) = torch.autograd.grad(lp, x, torch.ones_like(lp))
        assert lp[:3].isnan().all() and float(lp[3].detach()) <= 0 and bool((grad[:3] == 0).all()) and bool((grad[3] != 0).any())
        with pytest.raises(IndexError):
            trl_amd.check_device_errors()


def test_unfiltered_scores_are_the_log_softmax():
    import trl_amd

    logits, _ = make_logits(64, 5003, "bf16", 171)
    ids = torch.randint(0, 5003, (64,), generator=torch.Generator().manual_seed(1))
    a = trl_amd.filtered_logps(logits.to(DEV), ids.to(DEV))
    b = trl_amd.selective_log_softmax(logits.to(DEV), ids.to(DEV), out_dtype=torch.float32)
    torch.testing.assert_close(a, b, atol=1e-5, rtol=0)


def test_what_is_drawn_scores_the_same():
    import trl_amd

    logits, u = make_logits(128, 8001, "bf16", 181)
    for s in FILTERS:
        ids, lp = trl_amd.sample_tokens(logits.to(DEV), u.to(DEV), **s)
        assert torch.equal(trl_amd.filtered_logps(logits.to(DEV), ids, **s), lp)


def test_refusals():
    import trl_amd

    x, u = torch.randn(3, 50, device=DEV), torch.rand(3, device=DEV)
    ids = torch.zeros(3, dtype=torch.long, device=DEV)
    for bad in (dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf), dict(temperature=1e-320), dict(top_p=0.0),
                dict(top_p=1.5), dict(top_p=math.nan), dict(min_p=-0.1), dict(min_p=1.1), dict(top_p=torch.ones(4, device=DEV)),
                dict(row_mask=torch.ones(4, device=DEV))):
        with pytest.raises(ValueError):
            trl_amd.sample_tokens(x, u, **bad)
        with pytest.raises(ValueError):
            trl_amd.filtered_logps(x, ids, **bad)
    with pytest.raises(ValueError):
        trl_amd.sample_tokens(x, u[:2])
    with pytest.raises(ValueError):
        trl_amd.filtered_logps(x, ids[:2])
    with pytest.raises(TypeError):
        trl_amd.sample_tokens(x.double(), u)
    with pytest.raises(RuntimeError):
        trl_amd.sample_tokens(x, u.cpu())
    with pytest.raises((RuntimeError, NotImplementedError)):
        trl_amd.sample_tokens(x.cpu(), u.cpu())
    ids, lp = trl_amd.sample_tokens(x[:0], u[:0])
    assert ids.shape == lp.shape == (0,)
    with pytest.raises(RuntimeError):  # the gradient's own gradient
        y = x.clone().requires_grad_(True)
        lp = trl_amd.filtered_logps(y, torch.zeros(3, dtype=torch.long, device=DEV))
        (g,) = torch.autograd.grad(lp.sum(), y, create_graph=True)
        g.sum().backward()
    assert not trl_amd.sample_tokens(x.requires_grad_(True), u)[1].requires_grad


def test_another_stream_and_a_captured_graph():
    import trl_amd

    logits, u = make_logits(20, 6001, "bf16", 191)
    x, v = logits.to(DEV), u.to(DEV)
    s = settings(0.9, 30, 0.9)
    want = trl_amd.sample_tokens(x, v, **s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = trl_amd.sample_tokens(x, v, **s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    static_x, static_u = x.clone().requires_grad_(True), v.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ids, lp = trl_amd.sample_tokens(static_x, static_u, **s)
        scored = trl_amd.filtered_logps(static_x, ids, **s)
        (grad,) = torch.autograd.grad(scored, static_x, torch.ones_like(scored))
    for seed in (192, 193, 194):
        logits, u = make_logits(20, 6001, "bf16", seed)
        with torch.no_grad():
            static_x.copy_(logits)
            static_u.copy_(u)
        graph.replay()
        torch.cuda.synchronize()
        y = logits.to(DEV).requires_grad_(True)
        want_ids, want = trl_amd.sample_tokens(y, u.to(DEV), **s)
        assert torch.equal(ids, want_ids) and torch.equal(lp, want) and torch.equal(scored.detach(), want)
        (want_grad,) = torch.autograd.grad(trl_amd.filtered_logps(y, want_ids, **s), y, torch.ones_like(want))
        assert torch.equal(grad, want_grad)
        trl_amd.check_device_errors()


def test_traced_calls_have_the_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import trl_amd

    with FakeTensorMode():
        x = torch.empty(2, 3, 5000, dtype=torch.bfloat16, device=DEV)
        ids, lp = trl_amd.sample_tokens(x, torch.empty(2, 3, device=DEV), top_k=5)
        assert ids.shape == lp.shape == (2, 3) and ids.dtype == torch.int64 and lp.dtype == torch.float32
        assert trl_amd.filtered_logps(x, ids, top_p=0.9).shape == (2, 3)


def test_top_k_beyond_32_bits():
    """Values for each row as int64: those over any vocabulary keep all tokens, those under 0 switch the filter off."""
    import trl_amd

    logits, u = make_logits(6, 3001, "bf16", 231)
    x, v = logits.to(DEV), u.to(DEV)
    ks = torch.tensor([2**32 + 1, 2**40, 2**63 - 1, -(2**32) + 1, -(2**63), 7], device=DEV)
    ids, lp = trl_amd.sample_tokens(x, v, top_k=ks)
    scored = trl_amd.filtered_logps(x, ids, top_k=ks)
    for i, k in enumerate((0, 0, 0, 0, 0, 7)):
        want_id, want = trl_amd.sample_tokens(x[i], v[i], top_k=k)
        assert ids[i] == want_id and lp[i] == want and scored[i] == want
    trl_amd.check_device_errors()
    with pytest.raises(RuntimeError):
        trl_amd.sample_tokens(x, v, top_k=ks.cpu())
    with pytest.raises(RuntimeError):
        trl_amd.filtered_logps(x, ids, row_mask=torch.ones(6, dtype=torch.bool))


def test_two_graphs_replayed_at_once():
    """Two captured calls of different sizes on two streams, replayed side by side: neither touches what the other works with."""
    import trl_amd

    made, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed, (rows, V, dtype, s) in ((241, (90, 50257, "bf16", settings(1.0, 0, 0.95))), (242, (40, 32000, "fp32", settings(0.8, 40, 0.9)))):
        logits, u = make_logits(rows, V, dtype, seed)
        x, v = logits.to(DEV), u.to(DEV)
        want = trl_amd.sample_tokens(x, v, **s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ids, lp = trl_amd.sample_tokens(x, v, **s)
        made.append((graph, ids, lp, want, x, v))
    for _ in range(5):
        for _, ids, lp, *_ in made:
            ids.fill_(-7)
            lp.fill_(-7.0)
        for stream, (graph, *_) in zip(streams, made):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
        for stream in streams:
            torch.cuda.current_stream().wait_stream(stream)
        for _, ids, lp, want, *_ in made:
            assert torch.equal(ids, want[0]) and torch.equal(lp, want[1])
    trl_amd.check_device_errors()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows", [1, 20, 63, 530])
def test_rows_of_very_many_candidates_side_by_side(rows, dtype):
    """Nuclei of thousands of tokens: as many as all CUs pass over together, more, and so many rows that none is; with short nuclei between
    them, a border among equal logits, and min-p beside top-p."""
    import trl_amd

    V = 9001 if rows > 1 else 50257
    logits, u = make_logits(rows, V, dtype, 250 + rows, slope=0.5)
    logits[::5] *= 6.0  # short nuclei
    if rows > 3:
        logits[3] = 1.5  # equal logits
        logits[2, : V // 2] = 2.0
    for s in (settings(0.9, 0, 0.9), settings(1.0, 0, 0.97, 0.02), settings(1.2, 0, 1.0, 1e-3)):
        check_draw(logits, u, s)
        x = logits.to(DEV)
        ids, lp = trl_amd.sample_tokens(x, u.to(DEV), **s)
        for _ in range(3):
            again = trl_amd.sample_tokens(x, u.to(DEV), **s)
            assert torch.equal(again[0], ids) and torch.equal(again[1], lp)
        assert torch.equal(trl_amd.filtered_logps(x, ids, **s), lp)
        one = trl_amd.sample_tokens(x[rows - 1], u[rows - 1].to(DEV), **s)
        assert one[0] == ids[rows - 1] and one[1] == lp[rows - 1]


def test_a_border_between_two_distant_tokens():
    """The nucleus ends where the next token lies far below the last one, and its mass is within 1e-5 of top_p on one side or the other:
    thousands of tokens of little mass follow."""
    import trl_amd

    V, heads = 20000, 12
    g = torch.Generator().manual_seed(271)
    x = torch.full((40, V), -3.0) + 0.5 * torch.rand(40, V, generator=g)
    for i in range(40):
        x[i, torch.randperm(V, generator=g)[:heads]] = torch.linspace(7.0, 1.0, heads) + 0.3 * torch.rand(heads, generator=g)
    u = torch.rand(40, generator=g)
    order = x.double().sort(-1, descending=True).values
    mass = order.softmax(-1).cumsum(-1)
    for at, off in ((heads - 1, 1e-6), (heads - 1, -1e-6), (heads - 2, 1e-5), (heads - 2, -1e-5), (5, 3e-5), (5000, 0.0)):
        p = (mass[:, at] + off).float()
        check_draw(x, u, settings(1.0, 0, p))
        ids, lp = trl_amd.sample_tokens(x.to(DEV), u.to(DEV), top_p=p.to(DEV))
        assert torch.equal(trl_amd.filtered_logps(x.to(DEV), ids, top_p=p.to(DEV)), lp)


@pytest.mark.parametrize("rows", [3, 515])
def test_nuclei_of_almost_everything(rows):
    """top_p so near 1 that the border lies among the last tokens, in rows of very many, with and without min-p and masked rows; ids outside
    the vocabulary are reported by such rows as well."""
    import trl_amd

    V = 6007
    logits, u = make_logits(rows, V, "fp32", 280, slope=0.4)
    for s in (settings(1.0, 0, 0.99995), settings(0.8, 0, 1.0 - 2.0**-24), settings(1.0, 0, 0.99999, 1e-3), settings(5.0, 0, 0.5), settings(40.0, 0, 0.999)):
        check_draw(logits, u, s)
    x, ids = logits.to(DEV), torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(281)).to(DEV)
    mask = torch.ones(rows, dtype=torch.bool, device=DEV)
    mask[1] = False
    s = settings(1.0, 0, 0.99)
    whole = trl_amd.filtered_logps(x, ids, **s)
    part = trl_amd.filtered_logps(x, ids, row_mask=mask, **s)
    assert part[1] == 0 and torch.equal(part[mask], whole[mask])
    trl_amd.check_device_errors()
    ids[2] = V
    assert torch.isnan(trl_amd.filtered_logps(x, ids, **s)[2])
    with pytest.raises(IndexError):
        trl_amd.check_device_errors()


def test_very_many_candidates_of_a_large_vocabulary():
    import trl_amd

    V = trl_amd._lib.lib.trlk_token_filter_max_vocab()
    logits, u = make_logits(2, V, "bf16", 291, slope=0.3)
    check_draw(logits, u, settings(1.0, 0, 0.9))
    check_draw(logits, u, settings(1.0, 0, 1.0, 0.05))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_a_top_k_of_a_thousand_and_more(dtype):
    logits, u = make_logits(5, 20011, dtype, 301)
    logits[4] = logits[4].sign()  # three values
    for k in (900, 1024, 1025, 1500, 2500, 4095, 4097, 19999):
        for s in (settings(1.0, k), settings(0.7, k, 0.9), settings(3.0, k, 0.999, 1e-3)):
            check_draw(logits, u, s)


@pytest.mark.parametrize("shape", [(0,), (3, 0), (0, 4), (2, 3, 0), (2, 0, 3), (0, 2, 3), (2, 0, 3, 4), (2, 3, 4, 0), (2, 1, 3, 2)])
def test_ranks_and_no_rows(shape):
    """Leading dimensions of any number and size, zero among them."""
    import trl_amd

    g = torch.Generator().manual_seed(5)
    x = torch.randn(*shape, 70, generator=g).to(DEV).requires_grad_()
    u = torch.rand(shape, generator=g).to(DEV)
    s = settings(0.8, 9, 0.9)
    ids, logps = trl_amd.sample_tokens(x, u, **s)
    assert ids.shape == logps.shape == shape and ids.dtype == torch.int64
    scored = trl_amd.filtered_logps(x, ids, **s)
    assert scored.shape == shape and torch.equal(scored.detach(), logps)
    scored.sum().backward()
    assert x.grad.shape == x.shape
    if x.numel():
        want, _ = expected(x, s, u)
        assert torch.equal(ids.cpu().reshape(-1), want)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_the_largest_temperatures_and_logits(dtype):
    """Logits of up to 3e38 and a temperature of up to 2^100: distances beyond fp32's range have no weight.  Larger temperatures of a row's own
    have no distribution."""
    import trl_amd

    g = torch.Generator().manual_seed(31)
    for V in (300, 6000):
        near = (torch.rand(6, V, generator=g) * 2.0**101 - 2.0**100).to(DTYPES[dtype])
        far = ((torch.rand(6, V, generator=g) * 2 - 1) * 3e38).to(DTYPES[dtype])
        far[::2, : V // 2] = 3e38
        u = torch.rand(6, generator=g)
        for logits in (near, far):
            for s in (settings(2.0**100), settings(2.0**100, 0, 0.9), settings(2.0**99, 0, 1.0, 0.3), settings(2.0**100, 0, 0.95, 0.2),
                      settings(2.0**100, 20, 0.9)):
                check_draw(logits, u, s)
        t = torch.tensor([2.0**100, 2.0**101, 3e38, 1.0, math.inf, 0.0], device=DEV)
        ids, lp = trl_amd.sample_tokens(near.to(DEV), u.to(DEV), t, 0, 0.9)
        with pytest.raises(ValueError, match="no distribution"):
            trl_amd.check_device_errors()
        assert (ids < 0).tolist() == [False, True, True, False, True, False] and torch.equal(lp.isnan(), ids < 0)


@pytest.mark.parametrize("V", [5, 3000])
def test_the_gradient_at_the_smallest_temperatures(V):
    """1 / T beyond fp32: where one token has all of the mass the gradient is 0, where two equal ones share it it is infinite, elsewhere 0."""
    import trl_amd

    for T in (1e-38, 1e-39, 1e-60, 1e-300):
        x = torch.linspace(-1, 1, V).repeat(3, 1)
        x[1, V - 2] = 1.0
        x = x.to(DEV).requires_grad_()
        for s in (settings(T), settings(T, 0, 0.9), settings(T, 3)):
            ids = torch.full((3,), V - 1, device=DEV)
            lp = trl_amd.filtered_logps(x, ids, **s)
            want = torch.tensor([0.0, -math.log(2.0), 0.0])
            assert bool(((lp.detach().cpu() - want).abs() <= 1e-6).all())
            (grad,) = torch.autograd.grad(lp, x, torch.tensor([100.0, 100.0, 0.0], device=DEV))
            grad = grad.cpu()
            assert not grad[0].any() and not grad[2].any() and not grad[1, :-2].any()
            assert grad[1, -1] == math.inf and grad[1, -2] == -math.inf


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows", [3, 515])
def test_min_p_ends_a_long_row_before_top_p(rows, dtype):
    """Thousands of tokens over min-p's border that hold less than top_p of the mass: the border is min-p's, and top-p's is not looked at."""
    import trl_amd

    V = 20000
    g = torch.Generator().manual_seed(rows)
    w = torch.where(torch.rand(rows, V, generator=g) < 0.3, 0.2 + 0.8 * torch.rand(rows, V, generator=g), 0.1 * (1 - 0.2 * torch.rand(rows, V, generator=g)))
    logits, u = w.log().to(DTYPES[dtype]), torch.rand(rows, generator=g)
    s = settings(1.0, 0, 0.95, 0.15)
    tokens, weights = row_support(logits[0].double(), 1.0, 0, 0.95, 0.15)
    assert len(tokens) > 4096 and float(weights.sum() / (logits[0].double() - logits[0].double().max()).exp().sum()) < 0.8
    check_draw(logits, u, s)
    ids, lp = trl_amd.sample_tokens(logits.to(DEV), u.to(DEV), **s)
    assert torch.equal(trl_amd.filtered_logps(logits.to(DEV), ids, **s), lp)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_top_p_of_equal_logits_at_a_border(dtype):
    """n equal logits, top_p a whole number of n-ths: exactly so many are kept, wherever the logits lie and whatever the temperature and the number
    of rows (a sum that is off in its last bits must not add one)."""
    import trl_amd

    for n, V in ((2, 2), (2, 500), (4, 7000), (8, 8), (64, 64), (256, 3000), (4096, 4096), (8192, 8192)):
        for rows in (1, 40, 520 if V < 1000 else 3):
            g = torch.Generator().manual_seed(n + rows)
            top = (torch.randn(rows, 1, generator=g) * 8).to(DTYPES[dtype])
            x = torch.full((rows, V), -math.inf, dtype=DTYPES[dtype])
            x[:, V - n :] = top
            t = 10.0 ** (4 * torch.rand(rows, generator=g) - 2)
            for part in (0.5, 0.25, 0.75):
                kept = max(1, int(part * n)) if part * n == int(part * n) else None
                if kept is None:
                    continue
                for u, place in ((0.0, 0), (1 - 2.0**-24, kept - 1)):
                    s = dict(temperature=t.to(DEV), top_p=part)
                    ids, lp = trl_amd.sample_tokens(x.to(DEV), torch.full((rows,), u, device=DEV), **s)
                    assert bool((ids == V - n + place).all()), (n, V, rows, part, u, ids.unique())
                    assert bool(((lp.double().cpu() + math.log(kept)).abs() <= 2.0**-24 * math.log(kept) + 1e-11).all())
                    assert torch.equal(trl_amd.filtered_logps(x.to(DEV), ids, **s), lp)
                out = torch.full((rows,), V - n + kept, device=DEV)
                assert bool((trl_amd.filtered_logps(x.to(DEV), out, **s) == -math.inf).all())
