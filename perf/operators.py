"""The work of the two ends of an on-policy training step, as cases that can be timed and compared: drawing a batch's next
tokens, scoring drawn tokens under the distribution they came from, and the optimiser's step.

A case is a dict of plain values; `prepare` makes what a program holds before the call, `run` is one pass, `work` what that
pass cannot do without, `exact` its result in 64 bits.  The kinds:

  sample   next tokens from the logits of a generation step and one given uniform number per row, with temperature, top-k,
           top-p and min-p, and their log-probs under the filtered distribution
  score    log-probs of given tokens under the filtered distribution, and the gradient of the logits
  adamw    one AdamW step over the tensors of a model or its adapters, with the global gradient norm clipped; both moments
           in fp32, or in 8 bits with one scale per 256 entries

A row's tokens are ordered by logit, ties by index.  Top-k keeps the first k of them, top-p those before which less than
top_p of the mass (that top-k kept) lies, min-p those whose probability is at least min_p times the largest; temperature 0
keeps the first.  A token is drawn by inverting the cumulative sum of the kept tokens in index order.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
VOCABS = (32000, 32001, 50257, 50264, 128256, 128257, 151665, 151936, 151937, 202048, 256000, 262144)
HIDDEN = (1024, 1536, 2048, 2560, 3584, 4096)
LARGEST_SAMPLE = 512 * 151936  # logits of the largest sample case
LARGEST_SCORE = 8 * 513 * 151936  # and of the largest score case
LARGEST_MODEL = 480e6  # entries of the largest optimiser case
BETA1, BETA2, EPS, WEIGHT_DECAY, LR, MAX_NORM = 0.9, 0.999, 1e-8, 0.01, 1e-4, 1.0
BLOCK = 256  # entries that share a scale
SEED = 1234  # of the rounding of 8-bit moments


def listed():
    return [
        # one sequence being generated, chat defaults: the smallest call, launches and latency only
        dict(name="sample_one", kind="sample", R=1, V=32000, dtype="bf16", temperature=0.7, top_k=50, top_p=0.95, min_p=0.0),
        # a step of on-policy generation with the trainer's defaults: temperature alone
        dict(name="sample_plain", kind="sample", R=64, V=151936, dtype="bf16", temperature=1.0, top_k=0, top_p=1.0, min_p=0.0),
        # nucleus sampling, a tokenizer that gained a token
        dict(name="sample_nucleus", kind="sample", R=256, V=128257, dtype="bf16", temperature=0.8, top_k=0, top_p=0.95, min_p=0.0),
        # a large batch of requests with settings of their own in fp32, some of them under a grammar's mask
        dict(name="sample_mixed", kind="sample", R=384, V=151936, dtype="fp32", temperature=-1.0, top_k=-1, top_p=-1.0, min_p=-1.0),
        # a micro-batch of a small run
        dict(name="score_small", kind="score", B=4, T=64, V=32000, dtype="bf16", temperature=1.0, top_k=50, top_p=1.0, min_p=0.0),
        # nucleus sampling on a vocabulary that is no multiple of the vector width
        dict(name="score_odd", kind="score", B=8, T=125, V=50257, dtype="fp32", temperature=0.9, top_k=0, top_p=0.95, min_p=0.0),
        # a training micro-batch on the headline benchmark's vocabulary, top-k and top-p together
        dict(name="score_large", kind="score", B=8, T=512, V=151936, dtype="bf16", temperature=1.0, top_k=20, top_p=0.8, min_p=0.0),
        # low-rank adapters of all projections, fp32: hundreds of small tensors
        dict(name="adamw_adapters", kind="adamw", rank=16, H=2048, layers=16, V=0, dtype="fp32", bits=32),
        # a small model in bf16 with fp32 moments
        dict(name="adamw_bf16", kind="adamw", rank=0, H=1024, layers=8, V=32000, dtype="bf16", bits=32),
        # a larger one in fp32
        dict(name="adamw_fp32", kind="adamw", rank=0, H=2048, layers=6, V=50257, dtype="fp32", bits=32),
        # 8-bit moments: adapters of odd rank in bf16
        dict(name="adamw8_adapters", kind="adamw", rank=13, H=3584, layers=12, V=0, dtype="bf16", bits=8),
        # and a larger model
        dict(name="adamw8_bf16", kind="adamw", rank=0, H=2048, layers=6, V=50257, dtype="bf16", bits=8),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _filters(rng):
    kind = rng.choice(("none", "k", "p", "kp", "min", "all"))
    return dict(temperature=rng.choice((1.0, 0.9, 0.7, 0.6)),
                top_k=rng.choice((20, 50, 64, 100)) if kind in ("k", "kp", "all") else 0,
                top_p=rng.choice((0.8, 0.9, 0.95)) if kind in ("p", "kp", "all") else 1.0,
                min_p=rng.choice((0.02, 0.05, 0.1)) if kind in ("min", "all") else 0.0)


def draw(rng):
    kind = rng.choice(("sample", "sample", "score", "adamw"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if kind == "sample":
        V = rng.choice(VOCABS)
        case = dict(kind=kind, R=_log_uniform(rng, 1, min(512, LARGEST_SAMPLE // V)), V=V, dtype=dtype)
        if rng.random() < 0.2:  # settings of their own
            return dict(case, temperature=-1.0, top_k=-1, top_p=-1.0, min_p=-1.0)
        return dict(case, **_filters(rng))
    if kind == "score":
        V, B = rng.choice(VOCABS), _log_uniform(rng, 1, 16)
        most = LARGEST_SCORE // (B * V * (2 if dtype == "fp32" else 1)) - 1
        return dict(kind=kind, B=B, T=min(_log_uniform(rng, 24, 2048), most), V=V, dtype=dtype, **_filters(rng))
    bits = rng.choice((8, 32))
    if rng.random() < 0.4:
        return dict(kind=kind, rank=rng.choice((4, 8, 13, 16, 32)), H=rng.choice(HIDDEN), layers=_log_uniform(rng, 2, 32), V=0,
                    dtype=dtype, bits=bits)
    H, V = rng.choice(HIDDEN[:4]), rng.choice(VOCABS[:4])
    most = int((LARGEST_MODEL - V * H) // (11 * H * H))
    return dict(kind=kind, rank=0, H=H, layers=min(_log_uniform(rng, 1, 12), max(1, most)), V=V, dtype=dtype, bits=bits)


# ---------------------------------------------------------------------------------------------- inputs
def _shapes(case):
    """Shapes of a decoder's weights (square query and output projections, a quarter of the heads for keys and values, an
    MLP of 2.5 times the width, two norms per layer), or of low-rank adapters on its projections."""
    H, layers, V, rank = case["H"], case["layers"], case["V"], case["rank"]
    inner = 5 * H // 2
    projections = [(H, H), (H // 4, H), (H // 4, H), (H, H), (inner, H), (inner, H), (H, inner)]
    if rank:
        return [s for _ in range(layers) for o, i in projections for s in ((rank, i), (o, rank))]
    return [(V, H)] + [s for _ in range(layers) for s in projections + [(H,), (H,)]] + [(H,)]


def _lengths(B, T):
    """Completion lengths of a batch, 1/16 of the longest to the longest."""
    return [max(1, round(T / 16 + (T - T / 16) * (i + 1) / B)) for i in range(B)]


def _logits(rows, V, dtype, gd):
    """Logits whose sorted probabilities fall off as a power of the rank, with an exponent of 1.2 (an open question) to 3 (a
    nearly certain token) of the row's own: exponential numbers have that property."""
    out = torch.empty((rows, V), dtype=dtype, device=DEVICE)
    step = max(1, (1 << 28) // V)
    for i in range(0, rows, step):
        x = torch.empty((min(step, rows - i), V), device=DEVICE).exponential_(generator=gd)
        slope = 1.2 + 1.8 * torch.rand((x.shape[0], 1), generator=gd, device=DEVICE)
        out[i : i + step] = (x * slope - 4.0).to(dtype)
    return out


def _settings(case, rows, gd):
    """The filters of a batch: numbers, or (-1) a tensor with a value for each row."""
    if case["temperature"] >= 0:
        return {k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")}
    pick = lambda values, dtype: torch.tensor(values, dtype=dtype, device=DEVICE)[  # noqa: E731
        torch.randint(0, len(values), (rows,), generator=gd, device=DEVICE)]
    return dict(temperature=pick([0.0, 0.6, 0.7, 0.8, 1.0], torch.float32), top_k=pick([0, 0, 20, 50], torch.int32),
                top_p=pick([1.0, 0.8, 0.9, 0.95], torch.float32), min_p=pick([0.0, 0.0, 0.05], torch.float32))


def _flat(sizes, dtype):
    """One zeroed buffer, and a view of it for each size, at whole blocks."""
    whole = [-(-n // BLOCK) * BLOCK for n in sizes]
    flat = torch.zeros(sum(whole), dtype=dtype, device=DEVICE)
    at = [sum(whole[:i]) for i in range(len(whole))]
    return flat, [flat[a : a + n] for a, n in zip(at, sizes)]


def _prepare_adamw(case, gd):
    shapes, dtype = _shapes(case), DTYPES[case["dtype"]]
    sizes = [math.prod(s) for s in shapes]
    state = dict(kind="adamw", bits=case["bits"])
    for name, kind in (("p", dtype), ("g", dtype), ("m", torch.float32), ("v", torch.float32)):
        flat, views = _flat(sizes, kind)
        state["flat_" + name], state[name] = flat, [t.view(s) for t, s in zip(views, shapes)]
    scale = 10.0 ** (-4.5 + torch.rand(len(sizes), generator=gd, device=DEVICE))  # a tensor's gradients' size
    for i, n in enumerate(sizes):
        p, g, m, v = (state[k][i] for k in "pgmv")
        p.normal_(0.0, 0.02, generator=gd)
        m.normal_(0.0, 1.0, generator=gd).mul_(0.3 * scale[i])
        v.exponential_(generator=gd).mul_(scale[i] ** 2)
        g.copy_(torch.randn(p.shape, generator=gd, device=DEVICE).mul_(scale[i]))
    state["steps"] = list(torch.full((len(sizes),), 100.0, device=DEVICE).unbind())
    if case["bits"] == 8:
        zero = torch.zeros((), dtype=torch.int64, device=DEVICE)
        for name, kind in (("m", torch.float8_e4m3fn), ("v", torch.uint8)):
            codes, views = _flat(sizes, torch.uint8)
            scales = torch.ones(codes.numel() // BLOCK, device=DEVICE)
            scale_views = scales.split([-(-n // BLOCK) for n in sizes])
            for x, code, s in zip(state[name], views, scale_views):
                q, s[:] = _encode(x, name == "m", zero)
                code.copy_(q)
            state["flat_" + name], state[name] = codes.view(kind), [c.view(kind).view(s) for c, s in zip(views, shapes)]
            state["flat_%s_scale" % name], state[name + "_scale"] = scales, scale_views
    return state


def prepare(case, seed):
    gd = torch.Generator(device=DEVICE).manual_seed(seed)
    kind = case["kind"]
    if kind == "adamw":
        return _prepare_adamw(case, gd)
    V, dtype = case["V"], DTYPES[case["dtype"]]
    if kind == "sample":
        R = case["R"]
        logits = _logits(R, V, dtype, gd)
        if case["temperature"] < 0:  # every eighth request is bound to a grammar: about one token in a hundred is allowed
            logits[::8].masked_fill_(torch.rand((-(-R // 8), V), generator=gd, device=DEVICE) > 0.01, -math.inf)
        return dict(kind=kind, logits=logits, uniforms=torch.rand((R,), generator=gd, device=DEVICE), **_settings(case, R, gd))
    B, T = case["B"], case["T"]
    logits = _logits(B * T, V, dtype, gd).view(B, T, V)
    # tokens drawn from that distribution are mostly among the leading ones; one in some hundred lies outside the support
    leading = logits.topk(16, dim=-1).indices
    at = torch.empty((B, T, 1), device=DEVICE).exponential_(0.6, generator=gd).long().clamp_(max=15)
    ids = leading.gather(-1, at).squeeze(-1)
    other = torch.randint(0, V, (B, T), generator=gd, device=DEVICE)
    ids = torch.where(torch.rand((B, T), generator=gd, device=DEVICE) < 0.005, other, ids)
    lengths = torch.tensor(_lengths(B, T), device=DEVICE)[torch.randperm(B, generator=gd, device=DEVICE)]
    mask = torch.arange(T, device=DEVICE)[None] < lengths[:, None]
    upstream = torch.randn((B, T), generator=gd, device=DEVICE) * mask / mask.sum()
    return dict(kind=kind, logits=logits.requires_grad_(True), ids=ids, mask=mask, upstream=upstream, **_settings(case, 0, gd))


# ---------------------------------------------------------------------------------------------- plain forms
def _column(value, rows):
    """A setting as a 64-bit column, a value for each row."""
    value = torch.as_tensor(value, dtype=torch.float64, device=DEVICE).reshape(-1, 1)
    return value.expand(rows, 1)


def _kept_weights(x, s):
    """(weights of the kept tokens and 0 for the others, (x - max) / temperature), both 64-bit [rows, V]: a token's place
    beside a border and a sum over a vocabulary need them."""
    rows, V = x.shape
    temperature, top_k, top_p, min_p = (_column(s[k], rows) for k in ("temperature", "top_k", "top_p", "min_p"))
    top_k = torch.where(temperature == 0, 1.0, torch.where(top_k <= 0, float(V), top_k))
    temperature = torch.where(temperature == 0, 1.0, temperature)
    value, order = x.float().sort(dim=-1, descending=True, stable=True)
    z = (value.double() - value[:, :1].double()) / temperature
    kept = torch.arange(V, device=DEVICE) < top_k
    weight = torch.where(kept, z.exp(), 0.0)
    total = weight.sum(-1, keepdim=True)
    kept &= (weight.cumsum(-1) - weight < top_p * total) | (top_p >= 1)
    kept &= weight >= min_p
    weight = torch.where(kept, weight, 0.0)
    return torch.zeros_like(weight).scatter_(-1, order, weight), torch.empty_like(z).scatter_(-1, order, z)


def _plain_sample(s):
    weight, z = _kept_weights(s["logits"], s)
    cumulative = weight.cumsum(-1)
    total = cumulative[:, -1:]
    ids = (cumulative <= s["uniforms"].double()[:, None] * total).sum(-1)
    logps = z.gather(-1, ids[:, None]) - total.log()
    return ids, logps.squeeze(-1).float()


def _plain_score(s):
    B, T, V = s["logits"].shape
    x, ids, mask = s["logits"].detach().view(B * T, V), s["ids"].view(-1, 1), s["mask"].view(-1, 1)
    weight, z = _kept_weights(x, s)
    total = weight.sum(-1, keepdim=True)
    inside = weight.gather(-1, ids) > 0
    logps = torch.where(inside, z.gather(-1, ids) - total.log(), -math.inf)
    logps = torch.where(mask, logps, 0.0).view(B, T).float()
    g = torch.where(inside & mask, s["upstream"].view(-1, 1).double(), 0.0) / s["temperature"]
    grad = weight.mul_(-g / total).scatter_add_(-1, ids, g)
    return logps, grad.to(x.dtype).view(B, T, V)


def _mix(x):
    """A 32-bit hash of 32-bit whole numbers (held in 64 bits): xor with the upper half, multiply, twice."""
    x = ((x ^ (x >> 16)) * 0x55CE65AD) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0xCDBE2AF7) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random_bits(n, step, tensor):
    """32 bits for each of n entries, from the seed, the step's number, the tensor's place and the entry's."""
    salt = _mix(_mix(step.long() ^ SEED) + 0x9E3779B9 * (tensor + 1) & 0xFFFFFFFF)
    return _mix(salt + torch.arange(n, device=DEVICE) * 0x9E3779B1 & 0xFFFFFFFF)


def _encode(x, signed, bits):
    """8-bit codes and scales of fp32 `x`: 4 bits of exponent (bias 7), 3 of mantissa and a sign, or 4 and none, in units of
    a power of two for each block that takes its largest entry to at most 448; between two codes the given 16 random bits
    decide (0: downwards).  What is not zero keeps a code over zero where there is no sign: it is divided by."""
    n = x.numel()
    mantissa = 3 if signed else 4
    x = torch.nn.functional.pad(x.reshape(-1), (0, -n % BLOCK)).view(-1, BLOCK)
    largest = x.abs().amax(1)
    # the power of two, from the bits: 448 = 1.75 * 2^8
    word = largest.view(torch.int32)
    power = (word >> 23) - 127 - 8 + ((word & 0x7FFFFF) > 0x600000)
    power = power.clamp(-126, 127)
    scale = torch.where(largest > 0, ((power + 127) << 23).view(torch.float32), 1.0)
    y = (x.abs() / scale[:, None]).reshape(-1)[:n]
    word = y.view(torch.int32)
    shift = 23 - mantissa
    normal = ((word + (bits << (shift - 16))) >> shift) - (120 << mantissa)  # (the exponent's bias goes from 127 to 7)
    small = ((y * 2.0 ** (6 + mantissa + 16)).long() + bits) >> 16
    code = torch.where(y < 2.0**-6, small, normal)
    if signed:
        code = code | ((x.reshape(-1)[:n] < 0).long() << 7)
    else:
        code = torch.where(y > 0, code.clamp(min=1), code)
    return code.to(torch.uint8), scale


def _decode(code, scale, signed):
    """The fp32 values of codes."""
    n = code.numel()
    mantissa = 3 if signed else 4
    c = code.reshape(-1).view(torch.uint8).int()
    sign = torch.where(c > 127, -1.0, 1.0) if signed else 1.0
    c = c & 127 if signed else c
    value = torch.where(c < 2**mantissa, c.float() * 2.0 ** (-6 - mantissa), ((c + (120 << mantissa)) << (23 - mantissa)).view(torch.float32))
    return sign * value * scale.repeat_interleave(BLOCK)[:n]


def _plain_adamw_one(i, s, clip, eight):
    """One tensor's step in fp32, each product and sum rounded once."""
    p, g, step = s["p"][i], s["g"][i], s["steps"][i]
    step.add_(1.0)
    t = step.double()
    g = g.float().reshape(-1) * clip
    if eight:
        m, v = _decode(s["m"][i], s["m_scale"][i], True), _decode(s["v"][i], s["v_scale"][i], False)
    else:
        m, v = s["m"][i].reshape(-1), s["v"][i].reshape(-1)
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + g * g * (1 - BETA2)
    size = (LR / (1 - BETA1**t)).float()
    denominator = v.sqrt() * (1 / (1 - BETA2**t).sqrt()).float() + EPS
    p.copy_((p.float().reshape(-1) * (1 - LR * WEIGHT_DECAY) - size * (m / denominator)).view(p.shape))
    if eight:
        bits = _random_bits(g.numel(), step, i)
        code, s["m_scale"][i][:] = _encode(m, True, bits & 0xFFFF)
        s["m"][i].view(torch.uint8).copy_(code.view(p.shape))
        code, s["v_scale"][i][:] = _encode(v, False, bits >> 16)
        s["v"][i].copy_(code.view(p.shape))
    else:
        s["m"][i].copy_(m.view(p.shape))
        s["v"][i].copy_(v.view(p.shape))


def _plain_adamw(s):
    norm = torch.stack([g.double().square().sum() for g in s["g"]]).sum().sqrt()
    clip = (MAX_NORM / (norm + 1e-6)).clamp(max=1.0).float()
    [_plain_adamw_one(i, s, clip, s["bits"] == 8) for i in range(len(s["p"]))]
    return norm.float()


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    kind, s = state["kind"], state
    if kind == "sample":
        if not own:
            return _plain_sample(s)
        import trl_amd

        return trl_amd.sample_tokens(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                     min_p=s["min_p"])
    if kind == "score":
        if not own:
            return _plain_score(s)
        import trl_amd

        logps = trl_amd.filtered_logps(s["logits"], s["ids"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                       min_p=s["min_p"], row_mask=s["mask"])
        return logps.detach(), torch.autograd.grad(logps, s["logits"], s["upstream"])[0]
    eight = s["bits"] == 8
    if own:
        import trl_amd

        scales = dict(exp_avg_scales=s["m_scale"], exp_avg_sq_scales=s["v_scale"], seed=SEED) if eight else {}
        norm = trl_amd.adamw_step_(s["p"], s["g"], s["m"], s["v"], s["steps"], lr=LR, betas=(BETA1, BETA2), eps=EPS,
                                   weight_decay=WEIGHT_DECAY, max_grad_norm=MAX_NORM, **scales)
    else:
        norm = _plain_adamw(s)
    if not eight:
        return norm, s["flat_p"], s["flat_m"], s["flat_v"]
    # (both moments as the values that their codes stand for: 4 and 5 significant bits, exact in bf16)
    if own:
        m, v = (trl_amd.adamw_state_values(s["flat_" + k], s["flat_%s_scale" % k]) for k in "mv")
    else:
        m, v = (_decode(s["flat_" + k], s["flat_%s_scale" % k], k == "m").bfloat16() for k in "mv")
    return norm, s["flat_p"], m, v


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "sample":
        return {"bytes": case["R"] * (case["V"] * size + 32), "flops": 0}
    if case["kind"] == "score":  # the completions' rows are read, the gradient of all rows is written
        rows = case["B"] * case["T"]
        return {"bytes": (sum(_lengths(case["B"], case["T"])) + rows) * case["V"] * size + 24 * rows, "flops": 0}
    n = sum(math.prod(s) for s in _shapes(case))
    # parameter and moments read and written, gradient read; 8-bit moments also come back as bf16 values
    moments = 2 * 2 * 4 if case["bits"] == 32 else 2 * 2 * (1 + 4 / BLOCK) + 2 * 2
    return {"bytes": n * (3 * size + moments), "flops": 16 * n}


# ---------------------------------------------------------------------------------------------- in 64 bits
def _exact_row(x, temperature, top_k, top_p, min_p):
    """(kept tokens in index order, their probabilities) of one row of 64-bit logits."""
    if temperature == 0:
        top_k, temperature = 1, 1.0
    order = torch.argsort(-x, stable=True)
    if top_k > 0:
        order = order[:top_k]
    q = torch.softmax(x[order] / temperature, 0)
    n = 1 + int((torch.cumsum(q, 0)[:-1] < top_p).sum()) if top_p < 1 else q.numel()
    keep = (q >= min_p * q[0]) & (q > 0)
    keep[n:] = False
    tokens, at = order[keep].sort()
    q = q[keep][at]
    return tokens, q / q.sum()


def _exact_rows(s, rows):
    names = ("temperature", "top_k", "top_p", "min_p")
    each = [s[k].double().tolist() if torch.is_tensor(s[k]) else [s[k]] * rows for k in names]
    return [(t, int(k), p, m) for t, k, p, m in zip(*each)]


def _exact_sample(s):
    ids, logps = [], []
    for x, u, setting in zip(s["logits"], s["uniforms"], _exact_rows(s, s["logits"].shape[0])):
        tokens, q = _exact_row(x.double(), *setting)
        c = torch.cumsum(q, 0)
        at = torch.searchsorted(c, u.double() * c[-1], right=True)
        ids.append(tokens[at])
        logps.append(q[at].log())
    return torch.stack(ids), torch.stack(logps)


def _exact_score(s):
    B, T, V = s["logits"].shape
    settings = (s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    logps, grads = torch.zeros((B, T), dtype=torch.float64, device=DEVICE), torch.zeros((B, T, V), dtype=torch.float64, device=DEVICE)
    mask, ids = s["mask"].tolist(), s["ids"].tolist()
    logits = s["logits"].detach()
    for b in range(B):
        for t in range(T):
            if not mask[b][t]:
                continue
            tokens, q = _exact_row(logits[b, t].double(), *settings)
            p = torch.zeros(V, dtype=torch.float64, device=DEVICE).index_put_((tokens,), q)
            logps[b, t] = p[ids[b][t]].log()
            e = torch.zeros_like(p)
            e[ids[b][t]] = 1.0
            inside = (p[ids[b][t]] > 0).double()
            grads[b, t] = s["upstream"][b, t].double() * inside * (e - p) / s["temperature"]
    return logps, grads


def _exact_adamw(s, case):
    """The step from the definition.  The 8-bit moments have no value here: what is between two codes is settled by random
    bits, from the fp32 value."""
    total = sum(float(g.double().pow(2).sum()) for g in s["g"])
    norm = math.sqrt(total)
    clip = min(1.0, MAX_NORM / (norm + 1e-6))
    eight = case["bits"] == 8
    out = {k: torch.zeros(s["flat_" + k].shape, dtype=torch.float64, device=DEVICE) for k in "pmv"}
    at = 0
    for i, p in enumerate(s["p"]):
        n, t = p.numel(), float(s["steps"][i]) + 1
        if eight:
            m, v = _decode(s["m"][i], s["m_scale"][i], True).double(), _decode(s["v"][i], s["v_scale"][i], False).double()
        else:
            m, v = s["m"][i].double().flatten(), s["v"][i].double().flatten()
        g = s["g"][i].double().flatten() * clip
        m = BETA1 * m + (1 - BETA1) * g
        v = BETA2 * v + (1 - BETA2) * g**2
        update = (m / (1 - BETA1**t)) / ((v / (1 - BETA2**t)).sqrt() + EPS) + WEIGHT_DECAY * p.double().flatten()
        out["p"][at : at + n], out["m"][at : at + n], out["v"][at : at + n] = p.double().flatten() - LR * update, m, v
        at += -(-n // BLOCK) * BLOCK
    return torch.tensor(norm, dtype=torch.float64), out["p"], None if eight else out["m"], None if eight else out["v"]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(s)
    if case["kind"] == "score":
        return _exact_score(s) if case["B"] * case["T"] <= 4200 else None  # (a few milliseconds for each row)
    return _exact_adamw(s, case)
