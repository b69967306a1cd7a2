"""`patch_trl(adamw=True)` in a trainer's own loop on the GPU: created by it, stepped, saved and resumed from a checkpoint."""
import pytest
import torch

from test_optimizer_binding import fake_trl  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Model(torch.nn.Module):
    def __init__(self):
        super().__init__()
        torch.manual_seed(3)
        self.embed = torch.nn.Embedding(97, 64)
        self.body = torch.nn.Linear(64, 128)
        self.head = torch.nn.Linear(128, 97)

    def forward(self, ids, labels):
        logits = self.head(torch.nn.functional.gelu(self.body(self.embed(ids))))
        return {"loss": torch.nn.functional.cross_entropy(logits.flatten(0, 1), labels.flatten()), "logits": logits}


@pytest.mark.parametrize("optim", ["adamw_torch", "adamw_8bit"])
def test_a_trainer_makes_steps_saves_and_resumes(fake_trl, tmp_path, optim):  # noqa: F811
    import transformers

    import trl_amd
    from trl_amd import integration

    g = torch.Generator().manual_seed(5)
    data = [{"ids": torch.randint(0, 97, (12,), generator=g), "labels": torch.randint(0, 97, (12,), generator=g)} for _ in range(32)]
    assert integration.patch_trl(grpo=False, adamw=True) == 2
    try:
        def trainer(steps):
            args = transformers.TrainingArguments(output_dir=str(tmp_path), optim=optim, max_steps=steps, save_steps=3, learning_rate=1e-3,
                                                  per_device_train_batch_size=4, report_to=[], disable_tqdm=True, lr_scheduler_type="constant")
            return fake_trl["trl.trainer.grpo_trainer"].GRPOTrainer(model=Model(), args=args, train_dataset=data)

        whole = trainer(6)
        whole.train()
        opt = getattr(whole.optimizer, "optimizer", whole.optimizer)
        assert type(opt) is trl_amd.AdamW
        kinds = {n: opt.state[p]["exp_avg"].dtype for n, p in whole.model.named_parameters()}
        eight = torch.float8_e4m3fn if optim == "adamw_8bit" else torch.float32
        assert kinds["embed.weight"] == torch.float32 and kinds["body.weight"] == kinds["head.weight"] == eight
        resumed = trainer(6)
        resumed.train(resume_from_checkpoint=str(tmp_path / "checkpoint-3"))
        for (n, p), q in zip(whole.model.named_parameters(), resumed.model.parameters()):
            assert float(getattr(resumed.optimizer, "optimizer", resumed.optimizer).state[q]["step"]) == 6.0
            assert torch.equal(p, q), n
    finally:
        integration.unpatch_trl()
