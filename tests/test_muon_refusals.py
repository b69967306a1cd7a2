"""CPU-only checks of the orthogonalised updates' entry points: what they refuse is refused on the host, before anything is launched."""
import copy
import ctypes
import math

import pytest
import torch

FAKE = 0x1000  # never dereferenced: every call below fails validation first


class Matrix(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("param", "grad", "momentum")] + [
        ("rows", ctypes.c_int64), ("cols", ctypes.c_int64), ("dtype", ctypes.c_int32), ("group", ctypes.c_int32)]


class Group(ctypes.Structure):
    _fields_ = [(n, ctypes.c_double) for n in ("lr", "momentum", "weight_decay")] + [
        ("d_lr", ctypes.c_void_p), ("nesterov", ctypes.c_int32), ("adjust", ctypes.c_int32)]


def test_library_refuses():
    from trl_amd import _lib

    lib = _lib.lib

    def table(**changed):
        x = dict(param=FAKE, grad=FAKE, momentum=FAKE, rows=70, cols=130, dtype=_lib.BF16, group=0, **{})
        return (Matrix * 1)(Matrix(**{**x, **changed}))

    def step(x=None, n=1, groups=1, lr=0.1, momentum=0.9, decay=0.1, d_lr=None, adjust=0, steps=5, c=(3.4445, -4.775, 2.0315), eps=1e-7, ws=FAKE,
             ws_bytes=1 << 30):
        g = (Group * 1)(Group(lr, momentum, decay, d_lr, 1, adjust))
        return lib.trlk_muon_step(x if x is not None else table(), n, g, groups, steps, *c, eps, ws, ws_bytes, None)

    assert step(n=-1) == -1 and lib.trlk_muon_step(None, 1, None, 0, 5, 1.0, 0.0, 0.0, 1e-7, FAKE, 1 << 30, None) == -1
    for bad in (-0.1, 1.0, math.nan):
        assert step(momentum=bad) == -5 and "momentum" in _lib.last_error()
    assert step(lr=-1.0) == -5 and step(lr=math.nan) == -5 and step(decay=-1.0) == -5 and step(adjust=2) == -5
    assert step(table(group=1)) == -5 and step(table(group=-1)) == -5 and step(table(dtype=7)) == -3
    assert step(table(rows=-1)) == -2 and step(table(rows=32769, cols=32769)) == -2 and step(table(cols=(1 << 22) + 1)) == -2
    assert step(table(rows=32768, cols=1 << 20)) == -2
    for name in ("param", "grad", "momentum"):
        assert step(table(**{name: None})) == -1 and step(table(**{name: FAKE + 1})) == -4
    for bad in (0, -1, 101):
        assert step(steps=bad) == -5
    for bad in (0.0, -1.0, 2.0, 1e-31, math.nan):
        assert step(eps=bad) == -5
    for bad in ((math.inf, 0.0, 0.0), (9.0, 0.0, 0.0), (3.4445, 4.775, 2.0315), (1.0, 0.0, -8.0)):
        assert step(c=bad) == -5, bad
    need = lib.trlk_muon_workspace_bytes(table(), 1)
    assert need > 0 and step(ws_bytes=need - 1) == -6 and step(ws=None) == -6 and step(ws=FAKE + 16) == -6
    assert lib.trlk_muon_workspace_bytes(None, 1) == 0 and lib.trlk_muon_workspace_bytes(table(rows=-1), 1) == 0
    assert lib.trlk_muon_workspace_bytes(table(rows=0), 1) == 0
    assert step(table(rows=0, param=None, grad=None, momentum=None), ws=None, ws_bytes=0) == 0 and step(n=0, ws=None, ws_bytes=0) == 0
    assert lib.trlk_orthogonalize(table(), 1, 5, 3.4445, -4.775, 2.0315, 1e-7, FAKE, 1 << 30, None) == -5  # a momentum
    assert lib.trlk_orthogonalize(table(momentum=None), 1, 5, 3.4445, -4.775, 2.0315, 1e-7, FAKE, need - 1, None) == -6


def test_host_tensors_raise():
    import trl_amd

    x = [torch.zeros((4, 5))]
    with pytest.raises(NotImplementedError):
        trl_amd.muon_step_(x, x, x)
    with pytest.raises(NotImplementedError):
        trl_amd.orthogonalize(x[0])
    p = torch.nn.Parameter(torch.zeros((4, 5)))
    p.grad = torch.zeros((4, 5))
    with pytest.raises(RuntimeError, match="GPU"):
        trl_amd.Muon([p]).step()


def params():
    return [torch.nn.Parameter(torch.zeros(s)) for s in ((4, 5), (6, 3), (5,))]


def test_settings():
    import trl_amd

    p = params()
    for bad in (dict(lr=-1.0), dict(weight_decay=-1.0), dict(momentum=1.0), dict(momentum=-0.1), dict(eps=0.0), dict(ns_steps=0), dict(ns_steps=101),
                dict(ns_coefficients=(1.0,)), dict(adjust_lr_fn="x")):
        with pytest.raises(ValueError):
            trl_amd.Muon(p[:2], **bad)
        with pytest.raises(ValueError):
            trl_amd.Muon([dict(params=p[:2], **bad)])
    with pytest.raises(ValueError, match="adamw"):
        trl_amd.Muon(p)
    for bad in (dict(betas=(1.0, 0.9)), dict(adamw_eps=-1.0)):
        with pytest.raises(ValueError):
            trl_amd.Muon([dict(params=p, adamw=True, **bad)])
    opt = trl_amd.Muon(p[:2])
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=p[2:]))
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=p[2:], adamw=True))
    again = copy.deepcopy(opt)
    assert again.param_groups[1]["adamw"] and again.param_groups[0]["momentum"] == 0.95


def test_foreign_states_are_refused():
    import trl_amd

    def optimizer(adamw):
        p = params()
        return trl_amd.Muon([dict(params=p[:2]), dict(params=p[2:], adamw=adamw)] if adamw else p[:2])

    whole = optimizer(True)
    state = whole.state_dict()
    theirs = torch.optim.AdamW(params()[:2])
    for q in theirs.param_groups[0]["params"]:
        q.grad = torch.ones_like(q)
    theirs.step()
    with pytest.raises(ValueError, match="momentum_buffer"):
        optimizer(False).load_state_dict(theirs.state_dict())
    changed = copy.deepcopy(state)
    changed["param_groups"][1]["adamw"] = False
    with pytest.raises(ValueError, match="AdamW"):
        whole.load_state_dict(changed)
    muon = torch.optim.Muon(params()[:2])
    for q in muon.param_groups[0]["params"]:
        q.grad = torch.ones_like(q)
    muon.step()
    wrong = copy.deepcopy(muon.state_dict())
    wrong["state"][0]["momentum_buffer"] = torch.zeros((5, 4))
    with pytest.raises(ValueError, match="momentum_buffer"):
        optimizer(False).load_state_dict(wrong)
    mine = optimizer(False)
    mine.load_state_dict(muon.state_dict())
    q = mine.param_groups[0]["params"][0]
    assert mine.state[q]["momentum_buffer"].dtype == torch.float32 and mine.param_groups[0]["adamw"] is False


class Small(torch.nn.Module):
    def __init__(self, tied):
        super().__init__()
        self.embed = torch.nn.Embedding(11, 6)
        self.a, self.norm, self.lm_head = torch.nn.Linear(6, 6), torch.nn.LayerNorm(6), torch.nn.Linear(6, 11, bias=False)
        self.frozen = torch.nn.Linear(6, 6).requires_grad_(False)
        if tied:
            self.lm_head.weight = self.embed.weight

    def get_output_embeddings(self):
        return self.lm_head


def test_param_groups():
    import trl_amd

    for tied in (False, True):
        model = Small(tied)
        matrices, rest = trl_amd.muon_param_groups(model)
        assert [id(p) for p in matrices["params"]] == [id(model.a.weight)] and rest["adamw"]
        assert {id(p) for p in rest["params"]} == {id(p) for p in (model.embed.weight, model.a.bias, model.norm.weight, model.norm.bias, model.lm_head.weight)}
        trl_amd.Muon([matrices, rest], adjust_lr_fn="match_rms_adamw")


def test_convolutions_are_no_matrices():
    import trl_amd

    model = torch.nn.Sequential(torch.nn.Conv2d(3, 8, 4), torch.nn.Conv1d(8, 8, 4, groups=8), torch.nn.Linear(8, 8))
    matrices, rest = trl_amd.muon_param_groups(model)
    assert [id(p) for p in matrices["params"]] == [id(model[2].weight)] and len(rest["params"]) == 5


def test_shapes_for_tracers():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import trl_amd

    with FakeTensorMode():
        x = torch.empty((3, 50, 8), dtype=torch.bfloat16, device="cuda")
        assert trl_amd.orthogonalize(x).shape == x.shape and trl_amd.orthogonalize([x, x[0]])[1].shape == (50, 8)


@pytest.mark.parametrize("way", ["mine", "theirs"])
def test_loaded_moments_lie_as_their_parameters_do(way):
    """A convolution's weight with its channels last, a transposed matrix: AdamW's step asks for moments in the parameter's order."""
    import trl_amd

    conv = torch.nn.Conv2d(3, 8, 4).to(memory_format=torch.channels_last)
    turned = torch.nn.Parameter(torch.randn(6, 4).t())
    matrix = torch.nn.Parameter(torch.randn(5, 4))
    groups = [dict(params=[matrix]), dict(params=[conv.weight, turned], adamw=True)]
    opt = trl_amd.Muon(copy.deepcopy(groups))
    params = [p for g in opt.param_groups for p in g["params"]]
    fresh = [opt._state_of(p, i > 0) for i, p in enumerate(params)]
    gen = torch.Generator().manual_seed(0)
    for s in fresh:
        for t in s.values():
            t.copy_(torch.randn(t.shape, generator=gen))
    state = copy.deepcopy(opt.state_dict())
    if way == "theirs":  # (saved without their layout)
        state["state"] = {i: {k: t.contiguous() for k, t in s.items()} for i, s in state["state"].items()}
    again = trl_amd.Muon(copy.deepcopy(groups))
    again.load_state_dict(state)
    for p, s in zip((p for g in again.param_groups for p in g["params"]), fresh):
        assert set(again.state[p]) == set(s)
        for k, t in s.items():
            got = again.state[p][k]
            assert torch.equal(got, t) and got.dtype == torch.float32 and got.device == p.device
            assert k == "step" or got.stride() == p.stride() == t.stride(), k


class Wrapper(torch.nn.Module):
    """As a data-parallel wrapper has its model."""

    def __init__(self, module):
        super().__init__()
        self.module = module


def test_param_groups_of_wrapped_models_and_other_heads():
    import transformers

    import trl_amd

    for tied in (False, True):
        model = Small(tied)
        matrices, rest = trl_amd.muon_param_groups(Wrapper(Wrapper(model)))
        assert [id(p) for p in matrices["params"]] == [id(model.a.weight)]
        assert id(model.lm_head.weight) in {id(p) for p in rest["params"]}
    config = transformers.LlamaConfig(hidden_size=16, intermediate_size=32, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=2,
                                      vocab_size=50, num_labels=2, pad_token_id=0)
    for kind in (transformers.LlamaForCausalLM, transformers.LlamaForSequenceClassification, transformers.LlamaForTokenClassification,
                 transformers.LlamaForQuestionAnswering):
        for model in (kind(config), Wrapper(kind(config))):
            matrices, rest = trl_amd.muon_param_groups(model)
            names = {id(p): name for name, p in model.named_parameters()}
            assert len(matrices["params"]) == 7 and all(".layers." in names[id(p)] for p in matrices["params"])
            assert len(matrices["params"]) + len(rest["params"]) == len(names)


def test_numbers_of_steps_are_whole_and_small(monkeypatch):
    """2^32 + 5 is not 5, and neither is 5.9."""
    import trl_amd

    seen = []
    monkeypatch.setattr(trl_amd.ops, "orthogonalize", lambda *args: seen.append(args) or list(args[0]))
    monkeypatch.setattr(trl_amd.ops, "muon_step_", lambda *args: seen.append(args))
    x = [torch.zeros((4, 5))]
    for bad in (2**32 + 5, -(2**32) + 5, 0, 101):
        for call in (lambda: trl_amd.orthogonalize(x[0], ns_steps=bad), lambda: trl_amd.muon_step_(x, x, x, ns_steps=bad),
                     lambda: trl_amd.Muon([torch.nn.Parameter(x[0])], ns_steps=bad)):
            with pytest.raises(ValueError, match="ns_steps"):
                call()
    for call in (lambda: trl_amd.orthogonalize(x[0], ns_steps=5.9), lambda: trl_amd.muon_step_(x, x, x, ns_steps=5.9),
                 lambda: trl_amd.Muon([torch.nn.Parameter(x[0])], ns_steps=5.9)):
        with pytest.raises(TypeError):
            call()
    assert not seen
    trl_amd.orthogonalize(x[0], ns_steps=torch.tensor(100))
    assert seen[0][2] == 100
