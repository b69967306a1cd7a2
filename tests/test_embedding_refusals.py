"""CPU-only checks of the embedding's entry points: what they refuse is refused on the host, before anything is launched."""
import pytest
import torch

FAKE = 0x1000  # never dereferenced: every call below fails validation first


def test_library_refuses():
    from trl_amd import _lib

    def fwd(weight=FAKE, dtype=_lib.BF16, vocab=100, cols=64, stride=64, ids=FAKE, bits=64, n=10, out=FAKE):
        return _lib.lib.trlk_embedding_fwd(weight, dtype, vocab, cols, stride, ids, bits, n, 1.0, out, None, None)

    assert fwd(dtype=9) == -3 and fwd(bits=16) == -5 and fwd(n=-1) == -2 and fwd(vocab=-1) == -2 and fwd(cols=-1) == -2
    assert fwd(cols=(1 << 20) + 1, stride=1 << 21) == -2 and fwd(n=1 << 31) == -2 and fwd(vocab=(1 << 31) - 1) == -2
    assert fwd(stride=63) == -4 and fwd(weight=None) == -1 and fwd(ids=None) == -1 and fwd(out=None) == -1
    assert fwd(weight=FAKE + 1) == -4 and fwd(out=FAKE + 1) == -4 and fwd(ids=FAKE + 4) == -4
    assert fwd(n=0, weight=None) == 0 and fwd(cols=0, stride=0) == 0 and _lib.last_error() == ""

    def bwd(grad=FAKE, dtype=_lib.BF16, n=10, cols=64, stride=64, ids=FAKE, bits=64, vocab=100, add=1, dw=FAKE, out=_lib.BF16, out_stride=64,
            ws=FAKE, ws_bytes=1 << 20):
        return _lib.lib.trlk_embedding_bwd(grad, dtype, n, cols, stride, ids, bits, vocab, 1.0, -1, add, dw, out, out_stride, None, ws, ws_bytes, None)

    assert bwd(dtype=9) == -3 and bwd(out=_lib.F16) == -3 and bwd(dtype=_lib.F32) == -3 and bwd(bits=8) == -5
    assert bwd(n=-1) == -2 and bwd(n=1 << 31) == -2 and bwd(cols=(1 << 20) + 1, stride=1 << 21, out_stride=1 << 21) == -2
    assert bwd(stride=63) == -4 and bwd(out_stride=63) == -4 and bwd(out_stride=72, add=0) == -4
    assert bwd(grad=None) == -1 and bwd(ids=None) == -1 and bwd(dw=None) == -1
    assert bwd(grad=FAKE + 1) == -4 and bwd(dw=FAKE + 1) == -4 and bwd(ids=FAKE + 4) == -4
    need = _lib.lib.trlk_embedding_bwd_workspace_bytes(10, 100, 64)
    assert need > 0 and bwd(ws_bytes=need - 1) == -6 and bwd(ws=None) == -6 and bwd(ws=FAKE + 8) == -6
    assert _lib.lib.trlk_embedding_bwd_workspace_bytes(0, 100, 64) == 0 and _lib.lib.trlk_embedding_bwd_workspace_bytes(1 << 31, 100, 64) == 0
    assert bwd(n=0, grad=None, ids=None) == 0 and bwd(vocab=0, dw=None) == 0 and _lib.last_error() == ""


def test_host_tensors_and_bad_arguments_raise():
    import trl_amd

    ids, weight = torch.zeros((2, 3), dtype=torch.int64), torch.zeros((5, 4))
    with pytest.raises(NotImplementedError):
        trl_amd.embedding(ids, weight)
    with pytest.raises(NotImplementedError):
        trl_amd.embedding_grad_(weight, torch.zeros((2, 3, 4)), ids)
    for bad in (5, -6):
        with pytest.raises(ValueError, match="padding_idx"):
            trl_amd.embedding(ids, weight, padding_idx=bad)


class Model(torch.nn.Module):
    def __init__(self, embed):
        super().__init__()
        self.embed = embed

    def get_input_embeddings(self):
        return self.embed


class Other(torch.nn.Embedding):
    def forward(self, input):
        return super().forward(input) + 1


def test_patch_embedding_refuses():
    import trl_amd

    for module in (torch.nn.Linear(3, 4), torch.nn.Embedding(5, 4, max_norm=1.0), torch.nn.Embedding(5, 4, sparse=True),
                   torch.nn.Embedding(5, 4, scale_grad_by_freq=True), Other(5, 4)):
        with pytest.raises(ValueError):
            trl_amd.patch_embedding(Model(module))


def test_shapes_for_tracers():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import trl_amd

    with FakeTensorMode():
        weight = torch.empty((50, 8), dtype=torch.bfloat16, device="cuda")
        ids = torch.empty((2, 3), dtype=torch.int64, device="cuda")
        rows = trl_amd.embedding(ids, weight)
        assert rows.shape == (2, 3, 8) and rows.dtype == torch.bfloat16
        assert trl_amd.ops.embedding_bwd(rows, ids, 50, 1.0, -1).shape == (50, 8)


def scaled(name, **members):
    """A class whose name ends as those of transformers' scaled embeddings do, with their forward unless `members` has another."""
    def init(self, vocab, width, scale=3.0):
        torch.nn.Embedding.__init__(self, vocab, width)
        self.embed_scale = scale

    def forward(self, input_ids):
        return torch.nn.Embedding.forward(self, input_ids) * self.embed_scale

    return type(name + "ScaledWordEmbedding", (torch.nn.Embedding,), dict(dict(__init__=init, forward=forward), **members))


def test_patch_embedding_refuses_scaled_embeddings_that_do_more():
    import trl_amd
    from transformers.models.t5gemma2.modeling_t5gemma2 import T5Gemma2TextScaledWordEmbedding

    def one_token_more(self, input_ids):
        return torch.where(input_ids[..., None] == 7, 1.0, torch.nn.Embedding.forward(self, input_ids) * self.embed_scale)

    def shifted(self, input_ids):
        return torch.nn.Embedding.forward(self, input_ids) * self.embed_scale + 1.0

    def rooted(self, input_ids):
        return torch.nn.Embedding.forward(self, input_ids) * self.embed_scale**0.5

    for module in (T5Gemma2TextScaledWordEmbedding(11, 6, 0, embed_scale=2.0, eoi_token_index=5), scaled("OneMore", forward=one_token_more)(11, 6),
                   scaled("Shifted", forward=shifted)(11, 6), scaled("Rooted", forward=rooted)(11, 6)):
        with pytest.raises(ValueError, match="ScaledWordEmbedding"):
            trl_amd.patch_embedding(Model(module))
        assert "forward" not in vars(module)
    trl_amd.patch_embedding(Model(scaled("Plain")(11, 6)))


def test_scaled_embeddings_of_the_installed_models_are_known():
    import trl_amd
    from transformers.models.bart.modeling_bart import BartScaledWordEmbedding
    from transformers.models.gemma3.modeling_gemma3 import Gemma3TextScaledWordEmbedding

    for kind in (BartScaledWordEmbedding, Gemma3TextScaledWordEmbedding):
        for dtype in (torch.float32, torch.bfloat16):
            trl_amd.patch_embedding(Model(kind(11, 6, 3, embed_scale=33.941).to(dtype)))


def test_patch_embedding_refuses_a_forward_of_the_instance():
    """A hook of another library around the forward, for instance: it would be lost."""
    import trl_amd

    module = torch.nn.Embedding(5, 4)
    kept = module.forward

    def around(input):
        return kept(input) + 1

    module.forward = around
    with pytest.raises(ValueError, match="forward"):
        trl_amd.patch_embedding(Model(module))
    assert module.forward is around
    plain = Model(torch.nn.Embedding(5, 4))
    trl_amd.patch_embedding(plain)
    trl_amd.patch_embedding(plain)  # its own is not another's


def plain_embedding(input_ids, weight, *, scale=1.0, padding_idx=None):
    return (weight.float()[input_ids] * scale).to(weight.dtype)


def test_patched_modules_follow_their_scale(monkeypatch):
    """The model is cast, and its scale is changed, after the patch: the rows stay those of the module's own forward."""
    import sys

    import trl_amd
    from transformers.models.bart.modeling_bart import BartScaledWordEmbedding
    from transformers.models.gemma3.modeling_gemma3 import Gemma3TextScaledWordEmbedding

    monkeypatch.setattr(sys.modules["trl_amd.trainer.embedding"], "embedding", plain_embedding)
    ids = torch.arange(11).view(1, 11)
    for kind in (BartScaledWordEmbedding, Gemma3TextScaledWordEmbedding):
        torch.manual_seed(0)
        module = kind(11, 6, 0, embed_scale=1152**0.5)
        trl_amd.patch_embedding(Model(module))
        for dtype in (torch.float32, torch.bfloat16, torch.float32, torch.float16):
            module.to(dtype)
            for _ in range(2):
                assert torch.equal(module(ids), kind.forward(module, ids)), (kind, dtype)
        with torch.no_grad():
            module.embed_scale *= 0.5  # (a tensor in place)
        assert torch.equal(module(ids), kind.forward(module, ids))
        with torch.inference_mode():
            assert torch.equal(module(ids), kind.forward(module, ids))


def test_patched_modules_are_copied_and_pickled(monkeypatch):
    """Each copy reads its own table and can be patched again."""
    import copy
    import io
    import pickle
    import sys

    import trl_amd
    from transformers.models.gemma3.modeling_gemma3 import Gemma3TextScaledWordEmbedding

    monkeypatch.setattr(sys.modules["trl_amd.trainer.embedding"], "embedding", plain_embedding)
    ids = torch.arange(11).view(1, 11)

    def saved(model):
        file = io.BytesIO()
        torch.save(model, file)
        file.seek(0)
        return torch.load(file, weights_only=False)

    for module in (torch.nn.Embedding(11, 6), Gemma3TextScaledWordEmbedding(11, 6, 0, embed_scale=1152**0.5)):
        model = Model(module)
        trl_amd.patch_embedding(model)
        want = model.embed(ids)
        for way in (copy.deepcopy, lambda m: pickle.loads(pickle.dumps(m)), saved, lambda m: saved(copy.deepcopy(m))):
            other = way(model)
            with torch.no_grad():
                other.embed.weight.add_(1.0)
            assert torch.equal(model.embed(ids), want) and not torch.equal(other.embed(ids), want)
            assert torch.equal(other.to(torch.bfloat16).embed(ids), type(module).forward(other.embed, ids))
            trl_amd.patch_embedding(other)


def test_a_scale_that_requires_a_gradient_is_refused():
    import trl_amd

    ids, weight = torch.zeros((2, 3), dtype=torch.int64), torch.zeros((5, 4))
    scale = torch.tensor(2.0, requires_grad=True)
    with pytest.raises(ValueError, match="scale"):
        trl_amd.embedding(ids, weight, scale=scale)
    for taken in (scale.detach(), 2.0):  # (as far as the tensors, which are on the CPU)
        with pytest.raises(NotImplementedError):
            trl_amd.embedding(ids, weight, scale=taken)
    with torch.no_grad(), pytest.raises(NotImplementedError):
        trl_amd.embedding(ids, weight, scale=scale)
