"""The post-training path: the LM's scores of packed sequences, and the example that runs distillation, preference
tuning and policy updates on its head."""

import os
import sys

import pytest
import torch

from conftest import PKG_DIR


def test_next_token_labels():
    from kdn_b200.models.kernel_deltanet_lm import next_token_labels

    ids = torch.arange(10, 17)
    assert next_token_labels(ids, [0, 3, 4, 7]).tolist() == [11, 12, -100, -100, 15, 16, -100]
    assert next_token_labels(ids, torch.tensor([0, 7]), -1).tolist() == [11, 12, 13, 14, 15, 16, -1]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_score_matches_the_logits_of_every_prefix(dtype):
    """score() is the log-softmax of the head's logits in float64.  Both read the same logits: only the log-probability's
    fp32 arithmetic lies between (fp32 sums over 263 entries and exponents below 64: 2^-17 + 64 2^-23).  In chunks of 50
    rows the head runs another product kernel (kdn_linear has one for up to 64 rows), whose logits may differ by the
    2e-2 of the largest that the other comparison of two batch shapes here allows."""
    from kdn_b200.models import KernelDeltaNetLM

    torch.manual_seed(3)
    lm = KernelDeltaNetLM(vocab_size=263, d_model=128, num_layers=3, num_heads=2, d_ff=256, anchor_layers=[1])
    with torch.no_grad():
        for p in lm.parameters():
            if p.dim() == 2:
                p.normal_(std=1.0 / p.shape[1] ** 0.5)
    lm = lm.to("cuda", dtype)
    cu = [0, 70, 71, 204]
    ids = torch.randint(0, 263, (204,), generator=torch.Generator().manual_seed(1))
    got = lm.score(ids, cu, temperature=0.7)
    assert got.shape == (204,) and got.dtype == torch.float32
    logits = lm.lm_head(lm.hidden_states(ids, cu)).double()
    chunked = lm.score(ids, torch.tensor(cu), temperature=0.7, chunk_tokens=50)
    assert (got - chunked).abs().max() <= 2 * 2e-2 * logits.abs().max() / 0.7
    want = torch.log_softmax(logits / 0.7, -1)
    for i in range(3):
        s, e = cu[i], cu[i + 1]
        nxt = ids[s + 1:e].cuda()
        assert (got[s:e - 1].double() - want[torch.arange(s, e - 1), nxt]).abs().max() < 2 ** -17 + 64 * 2 ** -23 \
            if e - s > 1 else True
        assert got[e - 1] == 0
    # the rows that prefill reads are those of hidden_states
    cache = lm.new_cache(3, 204)
    last = lm.prefill(ids, cu, cache).double()
    assert (last - logits[[69, 70, 203]]).abs().max() <= 2e-2 * logits.abs().max()
    with pytest.raises(ValueError):
        lm.hidden_states(ids, [0, 70, 70, 204])
    with pytest.raises(ValueError):
        lm.score(ids, [0, 100])


@pytest.mark.gpu
def test_posttrain_example_learns():
    sys.path.insert(0, os.path.join(PKG_DIR, "examples"))
    import posttrain_head

    out = posttrain_head.main(steps=20, vocab=1003)
    first = lambda k: sum(out[k][:3]) / 3
    last = lambda k: sum(out[k][-3:]) / 3
    assert last("distillation loss") < 0.8 * first("distillation loss")
    assert abs(out["preference loss"][0] - 0.6931) < 1e-2  # log ratios start at zero
    assert last("preference loss") < 0.5 * first("preference loss")
    assert last("policy reward") > first("policy reward") + 0.05
