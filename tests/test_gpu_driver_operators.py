"""The language-model driver with --attention lsr and --max-grad-norm: a run end to end, and one step's
gradients of a small GPT-2 against the same model with the model library's attention."""
from __future__ import annotations

import copy
import json
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SMALL = "n_layer=2,n_embd=256,n_head=4,attn_pdrop=0"


def test_driver_with_both_operators(tmp_path):
    from lsr import lm_driver
    out = tmp_path / "run.json"
    argv = ["--muon-mode", "batched", "--init", "random", "--model-id", "gpt2", "--config-overrides", SMALL, "--steps", "3",
            "--warmup-steps", "1", "--seq-len", "130", "--grad-accum", "2", "--micro-batch", "2", "--attention", "lsr",
            "--max-grad-norm", "0.5", "--train-token-cache", str(tmp_path / "absent.pt"), "--train-cache-tokens", "100000",
            "--output", str(out)]
    assert lm_driver.main(argv) == 0
    s = json.loads(out.read_text())
    assert s["lsr"]["attention"] == "lsr" and s["lsr"]["max_grad_norm"] == 0.5
    assert math.isfinite(s["mean_measured_loss"])
    argv[argv.index(SMALL)] = SMALL.replace("attn_pdrop=0", "attn_pdrop=0.1")
    with pytest.raises(ValueError, match="attn_pdrop"):
        lm_driver.main(argv)


@pytest.mark.parametrize("padded", [False, True])
def test_model_gradients_with_either_attention(padded):
    """fp32. The two models differ in the order of fp32 sums alone; through two layers a gradient stays
    within 2^-12 of its tensor's norm (a few thousand roundings of 2^-24 each)."""
    from lsr import lm_driver as D
    from transformers import AutoModelForCausalLM
    cfg = D.model_config("gpt2", SMALL + ",embd_pdrop=0,resid_pdrop=0")
    torch.manual_seed(0)
    ours = AutoModelForCausalLM.from_config(cfg, attn_implementation=D._register_attention()).cuda().train()
    theirs = AutoModelForCausalLM.from_config(copy.deepcopy(cfg), attn_implementation="eager").cuda().train()
    theirs.load_state_dict(ours.state_dict())
    x = torch.randint(0, cfg.vocab_size, (2, 133), device="cuda")
    more, labels = {}, x
    if padded:
        more = {"attention_mask": (torch.arange(133, device="cuda") < torch.tensor([[133], [70]], device="cuda")).long()}
        labels = x.masked_fill(more["attention_mask"] == 0, -100)
    for m in (ours, theirs):
        m(input_ids=x, labels=labels, use_cache=False, **more).loss.backward()
    for (name, p), q in zip(ours.named_parameters(), theirs.parameters()):
        off = float((p.grad - q.grad).norm() / q.grad.norm().clamp(min=1e-20))
        assert off <= 2.0 ** -12, (name, off)
