"""GPU: what Trainer.token_logprobs leaves behind in the trainer.

Two passes over the same ids agree to TOL, the bound of every comparison of tensor-core results here: products round their operands to
tf32, whose step is 2^-10, so a difference of one fp32 rounding upstream (sums in another order) can move an operand x by 2^-10 |x|;
a logit is a sum of 128 products of size about 1 x 0.08, and of its operands only those next to a border move, by about 2^-10 x 0.08 = 8e-5 each."""

import numpy as np
import pytest
import torch

from tests.util import TOL, assert_close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["transformer", "decoder"])
def test_scoring_leaves_logits_and_disturbs_nothing(built, kind):
    """After scoring the output layer holds logits, after an inference pass probabilities again; a training step gives the
    same loss and gradients whether or not tokens were scored before it."""
    from opennn_b200 import trainer
    S_in, S_dec, V, B = 24, 16, 320, 4
    decoder_only = kind == "decoder"
    t = trainer.Trainer(trainer.DECODER_ONLY if decoder_only else trainer.TRANSFORMER, S_dec if decoder_only else S_in, S_dec, V, V, 128, 2, 256, 1, B)
    try:
        rng = np.random.default_rng(5)
        t.set_parameters((rng.standard_normal(t.parameters_number) * 0.08).astype(np.float32))
        gen = torch.Generator(device="cuda").manual_seed(6)
        dec, tgt = (torch.randint(1, V, (B, S_dec), generator=gen, device="cuda").float() for _ in range(2))
        enc = None if decoder_only else torch.randint(1, V, (B, S_in), generator=gen, device="cuda").float()
        tgt[2, 5:] = 0.0
        torch.cuda.synchronize()                              # the trainer has a stream of its own
        last = t.layers_number - 1

        before = t.step_device(dec, enc, tgt, update=False)
        gradients = t.get_gradients()
        t.forward(dec, enc, is_training=False)
        p = t.layer_output(last).reshape(-1, V).astype(np.float64)
        assert np.abs(p.sum(1) - 1).max() < 1e-5

        first = t.token_logprobs(dec, enc, tgt, top=3)
        logits = t.layer_output(last).reshape(-1, V).astype(np.float64)
        shifted = logits - logits.max(1, keepdims=True)
        softmax = np.exp(shifted) / np.exp(shifted).sum(1, keepdims=True)
        assert_close(softmax, p, TOL, "softmax of what scoring leaves")
        assert np.abs(logits.sum(1) - 1).max() > 0.1, "no longer probabilities"
        t.forward(dec, enc, is_training=False)
        assert_close(t.layer_output(last).reshape(-1, V), p, TOL, "probabilities again")

        second = t.token_logprobs(dec, enc, tgt, top=3)
        for a, b in [(first[k], second[k]) for k in (0, 1, 3)]:
            assert_close(a[tgt > 0].cpu().numpy(), b[tgt > 0].cpu().numpy(), TOL, "scores")
            assert torch.equal(a[tgt <= 0], b[tgt <= 0]), "padding"
        after = t.step_device(dec, enc, tgt, update=False)
        assert abs(after[0] - before[0]) <= TOL * abs(before[0]) and after[2] == before[2]
        assert_close(t.get_gradients(), gradients, TOL, "gradients")
    finally:
        t.close()
