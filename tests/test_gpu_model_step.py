"""The embedding, the fused head on the same table, and the optimiser of matrices and the rest, as a training step uses them together: against
the same model in 64 bits, and in a trainer's loop with a checkpoint resumed.

Tolerances.  The loss and the gradients pass through four products in fp32 (torch's) and the head's three-piece products: 2e-5 of their norms.  The
step is compared with its definition on the gradients that it was given, see test_gpu_muon."""
import copy

import pytest
import torch

from test_gpu_muon import check_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
VOCAB, WIDTH, INNER, PAD = 301, 96, 200, 7


class Block(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.norm = torch.nn.LayerNorm(WIDTH)
        self.up, self.down = torch.nn.Linear(WIDTH, INNER, bias=False), torch.nn.Linear(INNER, WIDTH, bias=False)

    def forward(self, x):
        return x + self.down(torch.nn.functional.gelu(self.up(self.norm(x))))


class Model(torch.nn.Module):
    """A decoder without its attention; the head is the embedding's table."""

    def __init__(self, tied=True):
        super().__init__()
        torch.manual_seed(5)
        self.embed = torch.nn.Embedding(VOCAB, WIDTH, padding_idx=PAD)
        self.blocks = torch.nn.ModuleList(Block() for _ in range(2))
        self.lm_head = torch.nn.Linear(WIDTH, VOCAB, bias=False)
        if tied:
            self.lm_head.weight = self.embed.weight

    def get_input_embeddings(self):
        return self.embed

    def get_output_embeddings(self):
        return self.lm_head

    def hidden(self, ids):
        x = self.embed(ids)
        for block in self.blocks:
            x = block(x)
        return x

    def forward(self, ids, labels):
        logits = self.hidden(ids) @ self.lm_head.weight.T
        return {"loss": torch.nn.functional.cross_entropy(logits.flatten(0, 1), labels.flatten()), "logits": logits}


def batch(seed, shape=(4, 33)):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, VOCAB, shape, generator=g)
    ids[:, -5:] = PAD
    return ids


def test_a_step_of_a_tied_model():
    import trl_amd

    model, exact = Model().to(DEV), Model().double()
    trl_amd.patch_embedding(model)
    opt = trl_amd.Muon(trl_amd.muon_param_groups(model), lr=0.02, weight_decay=0.1)
    assert [len(g["params"]) for g in opt.param_groups] == [4, 5]
    for step in range(3):
        ids = batch(step)
        mask = (ids != PAD).long()
        # labels of a causal model: position t is scored against token t + 1
        logps, _ = trl_amd.chunked_logprobs_from_hidden(model.hidden(ids.to(DEV)), model.lm_head.weight, ids.to(DEV), mask.to(DEV), 0.9, 128)
        loss = -(logps * mask[:, 1:].to(DEV)).sum() / mask[:, 1:].sum()
        opt.zero_grad()
        loss.backward()
        exact.load_state_dict({k: v.double().cpu() for k, v in model.state_dict().items()})
        logits = exact.hidden(ids)[:, :-1] @ exact.lm_head.weight.T / 0.9
        want = torch.log_softmax(logits, -1).gather(-1, ids[:, 1:, None]).squeeze(-1)
        want = -(want * mask[:, 1:]).sum() / mask[:, 1:].sum()
        exact.zero_grad()
        want.backward()
        assert abs(float(loss) - float(want)) <= 2e-5 * float(want)
        for (name, p), q in zip(model.named_parameters(), exact.parameters()):
            off = torch.linalg.vector_norm(p.grad.double().cpu() - q.grad)
            assert float(off) <= 2e-5 * float(torch.linalg.vector_norm(q.grad)) + 1e-9, name
        matrices = opt.param_groups[0]["params"]
        before = [[p.detach().clone() for p in matrices], [p.grad.clone() for p in matrices],
                  [opt.state[p]["momentum_buffer"].clone() if step else torch.zeros_like(p) for p in matrices]]
        others = [(p, p.detach().clone()) for p in opt.param_groups[1]["params"]]
        opt.step()
        check_step([p.detach() for p in matrices], [opt.state[p]["momentum_buffer"] for p in matrices], *before, lr=0.02, wd=0.1, beta=0.95,
                   nesterov=True, adjust=None)
        assert all(not torch.equal(p, q) for p, q in others)


def test_a_copy_of_the_model_reads_its_own_table():
    import trl_amd

    model = Model().to(DEV)
    trl_amd.patch_embedding(model)
    reference = copy.deepcopy(model)
    ids = batch(1).to(DEV)
    want = reference.embed(ids)
    with torch.no_grad():
        model.embed.weight.add_(1.0)
    assert torch.equal(reference.embed(ids), want) and not torch.equal(model.embed(ids), want)


def test_a_trainer_makes_steps_saves_and_resumes(tmp_path):
    import transformers

    import trl_amd

    data = [{"ids": batch(i, (1, 33))[0], "labels": batch(i + 100, (1, 33))[0]} for i in range(32)]

    def trainer():
        model = Model(tied=False).to(DEV)  # (the trainer's files hold no tensor twice)
        trl_amd.patch_embedding(model)
        opt = trl_amd.Muon(trl_amd.muon_param_groups(model), lr=1e-2, adjust_lr_fn="match_rms_adamw")
        args = transformers.TrainingArguments(output_dir=str(tmp_path), max_steps=6, save_steps=3, per_device_train_batch_size=4, report_to=[],
                                              disable_tqdm=True)
        return transformers.Trainer(model=model, args=args, train_dataset=data, optimizers=(opt, None)), model

    whole, model = trainer()
    whole.train()
    resumed, other = trainer()
    resumed.train(resume_from_checkpoint=str(tmp_path / "checkpoint-3"))
    for (name, p), q in zip(model.named_parameters(), other.named_parameters()):
        assert torch.equal(p, q[1]), name
