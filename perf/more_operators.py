"""The work of a training step before the first layer and behind the last gradient, as cases that can be timed and compared: the
embedding of the tokens with its gradient, and the optimiser's step for the matrices between embedding and head.

A case is a dict of plain values; `prepare` makes what a program holds before the call, `run` is one pass, `work` what that
pass cannot do without, `exact` its result in 64 bits.  The kinds:

  lookup         rows of the embedding table times a scale, as generation and a reference model's forward take them
  embed          the same in training: the rows, and the table's whole gradient (rows of the padding token get none)
  embed_add      the table's gradient added to one that is there, the tied head's for instance
  orthogonalize  matrices brought near the nearest matrix with orthonormal rows (or columns) by Newton-Schulz products
  muon           one optimiser step over a model's matrices or its adapters: momentum, the orthogonalised update, weight decay

With X = U / max(|U|, eps) (Frobenius norm; U transposed if it has more rows than columns), five times
  A = X X^T,  X = a X + (b A + c A A) X
is the orthogonalised U.  The step is
  m = momentum m + (1 - momentum) g,  U = momentum m + (1 - momentum) g,  p = p (1 - lr decay) - lr sqrt(max(1, rows / columns)) X
"""
import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
VOCABS = (32000, 32001, 50257, 50264, 128256, 128257, 151665, 151936, 151937, 202048, 256000, 262144)
HIDDEN = (1024, 1150, 1536, 2048, 2560, 3584, 4096)
LARGEST_TOKENS = 16 * 2048 * 4096  # entries of the largest batch of embedded tokens
LARGEST_TABLE = 151936 * 4096  # and of the largest table
LARGEST_STEP = 4 * 168 * 4096**3  # operations of the largest step's products: 168 H^3 for a layer of width H
STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
LR, MOMENTUM, WEIGHT_DECAY = 0.02, 0.95, 0.1
BLOCK = 256  # tensors of a list begin at whole blocks of so many entries


def listed():
    return [
        # the next token of one sequence: the smallest call, a launch and nothing else
        dict(name="lookup_one", kind="lookup", B=1, T=1, V=32000, H=1024, dtype="bf16", scaled=False),
        # the prompts and completions of a batch, scaled embeddings
        dict(name="lookup_batch", kind="lookup", B=16, T=2048, V=151936, H=4096, dtype="bf16", scaled=True),
        # a small run's micro-batch: a width and a vocabulary that are no multiples of a vector
        dict(name="embed_odd", kind="embed", B=8, T=125, V=50257, H=1150, dtype="fp16", scaled=False),
        # a training micro-batch of long completions
        dict(name="embed_large", kind="embed", B=16, T=2048, V=151936, H=4096, dtype="bf16", scaled=True),
        # a micro-batch of a small tied model in fp32
        dict(name="add_small", kind="embed_add", B=4, T=64, V=32000, H=1024, dtype="fp32", scaled=False),
        # a tied model with one of the largest vocabularies, the head's gradient being there
        dict(name="add_tied", kind="embed_add", B=8, T=1024, V=256000, H=2048, dtype="bf16", scaled=True),
        # one square projection
        dict(name="ortho_one", kind="orthogonalize", E=1, M=1024, N=1024, dtype="bf16"),
        # a layer's experts, wide and of odd sizes, in fp32
        dict(name="ortho_experts", kind="orthogonalize", E=24, M=1150, N=2816, dtype="fp32"),
        # low-rank adapters of all projections: hundreds of small matrices
        dict(name="muon_adapters", kind="muon", rank=16, H=2048, layers=16, dtype="fp32"),
        # a small model
        dict(name="muon_small", kind="muon", rank=0, H=1024, layers=8, dtype="bf16"),
        # a larger one in fp32
        dict(name="muon_fp32", kind="muon", rank=0, H=2048, layers=6, dtype="fp32"),
        # the widest: some layers of a 7 billion parameter model
        dict(name="muon_large", kind="muon", rank=0, H=4096, layers=4, dtype="bf16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("lookup", "embed", "embed", "embed_add", "orthogonalize", "muon", "muon"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if kind == "muon":
        if rng.random() < 0.4:
            return dict(kind=kind, rank=rng.choice((4, 8, 13, 16, 32, 64)), H=rng.choice(HIDDEN), layers=_log_uniform(rng, 2, 32), dtype=dtype)
        H = rng.choice(HIDDEN)
        most = int(LARGEST_STEP // (168 * H**3 * (3 if dtype == "fp32" else 1)))
        return dict(kind=kind, rank=0, H=H, layers=min(_log_uniform(rng, 1, 12), max(1, most)), dtype=dtype)
    if kind == "orthogonalize":
        M, N = _log_uniform(rng, 16, 4096), _log_uniform(rng, 16, 4096)
        m, n = min(M, N), max(M, N)
        most = int(min(LARGEST_STEP / 4 // (5 * (3 * m * m * n + m**3)), 2**29 // (m * n)))
        return dict(kind=kind, E=min(_log_uniform(rng, 1, 64), max(1, most)), M=M, N=N, dtype=dtype)
    V, H = rng.choice(VOCABS), rng.choice(HIDDEN)
    while V * H * (2 if dtype == "fp32" else 1) > LARGEST_TABLE:
        V, H = rng.choice(VOCABS), rng.choice(HIDDEN)
    tokens = min(_log_uniform(rng, 1, 32768), LARGEST_TOKENS // (H * (2 if dtype == "fp32" else 1)))
    B = min(_log_uniform(rng, 1, 64), tokens)
    return dict(kind=kind, B=B, T=max(1, tokens // B), V=V, H=H, dtype=dtype, scaled=rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------- inputs
def _shapes(case):
    """Shapes of a decoder's matrices (square query and output projections, a quarter of the heads for keys and values, an MLP of
    2.5 times the width), or of low-rank adapters on its projections."""
    H, rank = case["H"], case["rank"]
    inner = 5 * H // 2
    projections = [(H, H), (H // 4, H), (H // 4, H), (H, H), (inner, H), (inner, H), (H, inner)]
    layer = [s for o, i in projections for s in ((rank, i), (o, rank))] if rank else projections
    return layer * case["layers"]


def _lengths(B, T):
    """Lengths of a batch's sequences, 1/16 of the longest to the longest."""
    return [max(1, round(T / 16 + (T - T / 16) * (i + 1) / B)) for i in range(B)]


def _tokens(case, gd):
    """Token ids whose frequency falls off as one over the rank, behind the end of a sequence the padding token, which is the last
    one of the vocabulary."""
    B, T, V = case["B"], case["T"], case["V"]
    u = torch.rand((B, T), generator=gd, device=DEVICE, dtype=torch.float64)
    ids = ((V - 1) ** u).long().clamp_(1, V - 1) - 1
    ids = (ids * 7919 + 13) % (V - 1)
    if case["kind"] == "lookup":
        return ids
    lengths = torch.tensor(_lengths(B, T), device=DEVICE)[torch.randperm(B, generator=gd, device=DEVICE)]
    return torch.where(torch.arange(T, device=DEVICE) < lengths[:, None], ids, V - 1)


def _gradients(M, N, count, gd):
    """Matrices with a few large singular values and many small ones, as gradients have."""
    rank = max(1, min(M, N) // 8)
    size = torch.arange(1, rank + 1, device=DEVICE) ** -0.5
    left = torch.randn((count, M, rank), generator=gd, device=DEVICE)
    right = torch.randn((count, rank, N), generator=gd, device=DEVICE)
    return (left * size) @ right + torch.randn((count, M, N), generator=gd, device=DEVICE)


def _flat(shapes, dtype):
    """One zeroed buffer, and a view of it for each shape, at whole blocks."""
    whole = [-(-math.prod(s) // BLOCK) * BLOCK for s in shapes]
    flat = torch.zeros(sum(whole), dtype=dtype, device=DEVICE)
    return flat, [t[: math.prod(s)].view(s) for t, s in zip(flat.split(whole), shapes)]


def prepare(case, seed):
    gd = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    state = dict(kind=kind)
    if kind == "orthogonalize":
        x = torch.cat([_gradients(case["M"], case["N"], 1, gd) for _ in range(case["E"])])
        return dict(state, x=x.mul_(1e-4).to(dtype))
    if kind == "muon":
        shapes = _shapes(case)
        for name, held in (("p", dtype), ("g", dtype), ("m", torch.float32)):
            state["flat_" + name], state[name] = _flat(shapes, held)
        size = 10.0 ** (-4.5 + torch.rand(len(shapes), generator=gd, device=DEVICE))
        for i, (rows, columns) in enumerate(shapes):
            g = _gradients(rows, columns, 1, gd)[0].mul_(size[i])
            state["g"][i].copy_(g)
            state["m"][i].copy_(_gradients(rows, columns, 1, gd)[0].mul_(0.3 * size[i]).add_(g, alpha=0.3))
            state["p"][i].normal_(0.0, 0.02, generator=gd)
        return state
    B, T, V, H = (case[k] for k in "BTVH")
    state |= dict(ids=_tokens(case, gd), scale=math.sqrt(H) if case["scaled"] else 1.0, padding=V - 1)
    table = torch.empty((V, H), dtype=dtype, device=DEVICE).normal_(0.0, 0.02, generator=gd)
    if kind == "embed_add":
        state["grad"] = table.mul_(1e-3)
    else:
        state["table"] = table.requires_grad_(kind == "embed")
    if kind != "lookup":
        state["upstream"] = torch.empty((B, T, H), dtype=dtype, device=DEVICE).normal_(0.0, 1e-3, generator=gd)
    return state


# ---------------------------------------------------------------------------------------------- plain forms
def _plain_rows(s):
    return (s["table"].detach()[s["ids"]].float() * s["scale"]).to(s["table"].dtype)


def _plain_sums(s, into):
    """The upstream gradients of each token, added in fp32 to `into` [V, H]."""
    g = s["upstream"].flatten(0, 1).float() * s["scale"]
    g = torch.where((s["ids"] == s["padding"]).view(-1, 1), 0.0, g)
    return into.index_add_(0, s["ids"].view(-1), g)


def _plain_orthogonalized(x):
    """[E, M, N] fp32."""
    tall = x.shape[1] > x.shape[2]
    x = x.mT.contiguous() if tall else x
    norm = x.double().square().sum((1, 2), keepdim=True).sqrt().float()
    x = x / norm.clamp(min=EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        A = x @ x.mT
        x = a * x + (b * A + c * (A @ A)) @ x
    return x.mT if tall else x


def _plain_muon(s):
    """Matrices of one shape are stepped together."""
    by_shape = {}
    for i, p in enumerate(s["p"]):
        by_shape.setdefault(tuple(p.shape), []).append(i)
    for (rows, columns), each in by_shape.items():
        p, g, m = (torch.stack([s[k][i] for i in each]).float() for k in "pgm")
        m = MOMENTUM * m + (1 - MOMENTUM) * g
        x = _plain_orthogonalized(MOMENTUM * m + (1 - MOMENTUM) * g)
        p = p * (1 - LR * WEIGHT_DECAY) - LR * math.sqrt(max(1.0, rows / columns)) * x
        torch._foreach_copy_([s["m"][i] for i in each], list(m.unbind()))
        torch._foreach_copy_([s["p"][i] for i in each], list(p.unbind()))


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    kind, s = state["kind"], state
    if own:
        import trl_amd
    if kind == "lookup":
        return trl_amd.embedding(s["ids"], s["table"], scale=s["scale"]) if own else _plain_rows(s)
    if kind == "embed":
        if own:
            rows = trl_amd.embedding(s["ids"], s["table"], scale=s["scale"], padding_idx=s["padding"])
            return rows.detach(), torch.autograd.grad(rows, s["table"], s["upstream"])[0]
        table = s["table"]
        return _plain_rows(s), _plain_sums(s, torch.zeros(table.shape, device=DEVICE)).to(table.dtype)
    if kind == "embed_add":
        if own:
            trl_amd.embedding_grad_(s["grad"], s["upstream"], s["ids"], scale=s["scale"], padding_idx=s["padding"])
        else:
            s["grad"].copy_(_plain_sums(s, s["grad"].float() if s["grad"].dtype != torch.float32 else s["grad"]))
        return s["grad"]
    if kind == "orthogonalize":
        return trl_amd.orthogonalize(s["x"]) if own else _plain_orthogonalized(s["x"].float()).to(s["x"].dtype)
    if own:
        trl_amd.muon_step_(s["p"], s["g"], s["m"], lr=LR, momentum=MOMENTUM, nesterov=True, weight_decay=WEIGHT_DECAY,
                           ns_coefficients=COEFFICIENTS, ns_steps=STEPS, eps=EPS)
    else:
        _plain_muon(s)
    return s["flat_p"], s["flat_m"]


def _distinct(draws, V):
    """How many different tokens so many draws have, on average."""
    if draws == 1:
        return 1.0
    log_v = math.log(V - 1)
    return sum(1.0 - (1.0 - math.log1p(1.0 / i) / log_v) ** draws for i in range(1, V - 1))


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] in ("orthogonalize", "muon"):
        if case["kind"] == "muon":
            shapes = _shapes(case)
            each = 3 * size + 8  # parameter read and written, gradient read, momentum in fp32 read and written
        else:
            shapes = [(case["M"], case["N"])] * case["E"]
            each = 2 * size
        flops = 0
        for rows, columns in shapes:
            m, n = min(rows, columns), max(rows, columns)
            # X X^T and A A are symmetric: half of each
            flops += STEPS * (m * m * n + m**3 + 2 * m * m * n)
        return {"bytes": each * sum(math.prod(s) for s in shapes), "flops": flops}
    tokens, V, H = case["B"] * case["T"], case["V"], case["H"]
    if case["kind"] == "lookup":
        return {"bytes": (_distinct(tokens, V) + tokens) * H * size + 8 * tokens, "flops": 0}
    real = sum(_lengths(case["B"], case["T"]))
    rows = _distinct(real, V)
    if case["kind"] == "embed":  # table rows read, embedded tokens written, their gradients read, the table's gradient written
        return {"bytes": (rows + 1 + tokens + real + V) * H * size + 8 * tokens, "flops": real * H}
    return {"bytes": (real + 2 * rows) * H * size + 8 * tokens, "flops": real * H}


# ---------------------------------------------------------------------------------------------- in 64 bits
def _exact_orthogonal(u):
    """Of one matrix in 64 bits.  X = U h(U^T U) with U^T U (or U U^T) the smaller one: each iteration multiplies by its
    polynomial's factor, which is summed by Horner's rule."""
    x = u / max(float(torch.linalg.vector_norm(u)), EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        if x.shape[0] <= x.shape[1]:
            gram = x @ x.t()
            inner = c * gram
            inner.diagonal().add_(b)
            factor = gram @ inner
            factor.diagonal().add_(a)
            x = factor @ x
        else:
            gram = x.t() @ x
            inner = c * gram
            inner.diagonal().add_(b)
            factor = inner @ gram
            factor.diagonal().add_(a)
            x = x @ factor
    return x


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "orthogonalize":
        return torch.stack([_exact_orthogonal(x.double()) for x in s["x"]])
    if kind == "muon":
        p, m = s["flat_p"].double(), s["flat_m"].double()
        at = 0
        for weight, g in zip(s["p"], s["g"]):
            n = g.numel()
            w, v = p[at : at + n].view(g.shape), m[at : at + n].view(g.shape)
            v += (g.double() - v) * (1 - MOMENTUM)
            update = _exact_orthogonal(v + (g.double() - v) * (1 - MOMENTUM))
            stretch = max(1.0, g.shape[0] / g.shape[1]) ** 0.5
            w -= LR * (WEIGHT_DECAY * w + stretch * update)
            at += -(-n // BLOCK) * BLOCK
        return p, m
    ids = s["ids"].reshape(-1)
    if kind != "lookup":
        kept = ids != s["padding"]
        g = s["upstream"].flatten(0, 1)[kept].double().mul_(s["scale"])
        total = s["grad"].double() if kind == "embed_add" else torch.zeros(s["table"].shape, dtype=torch.float64, device=DEVICE)
        total.index_put_((ids[kept],), g, accumulate=True)
    if kind == "embed_add":
        return total
    rows = torch.nn.functional.embedding(s["ids"], s["table"].detach().double()) * s["scale"]
    return rows if kind == "lookup" else (rows, total)
