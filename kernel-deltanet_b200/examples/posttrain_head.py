"""Post-training of a hybrid Kernel-DeltaNet LM's head, in the three steps that follow upcycling:

    1. distillation    from the largest logits of a teacher (its other mass is one more class);
    2. preference      tuning on pairs of packed answers, against the distilled model's own scores;
    3. policy          updates on sampled tokens with a clipped ratio, a KL term and an entropy bonus.

    python kernel-deltanet_b200/examples/posttrain_head.py [--steps N] [--vocab V] [--seed S]

The blocks are frozen: they run the serving prefill, which keeps no activations (bf16, libkdn).  The head's logits come
from kdn_linear, each loss returns its value and d loss / d logits in one pass, and the head's gradient is one product
with the hidden states.  Teacher, student and data are random; what the script shows is the calls, and that each
step's loss falls.
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from kdn_b200 import (KernelDeltaNetLM, distillation_loss_and_grad, policy_loss_and_grad,  # noqa: E402
                      preference_loss_and_grad, token_logprobs)
from kdn_b200.kernels import glue  # noqa: E402
from kdn_b200.models.kernel_deltanet_lm import next_token_labels  # noqa: E402


class Head:
    """fp32 master weight of the LM head with Adam; logits in bf16 through kdn_linear."""

    def __init__(self, lm: KernelDeltaNetLM, lr: float):
        self.lm = lm
        self.master = lm.lm_head.weight.detach().float().clone().requires_grad_()
        self.opt = torch.optim.Adam([self.master], lr=lr)

    def logits(self, hidden: torch.Tensor) -> torch.Tensor:
        return glue.linear(hidden, self.lm.lm_head.weight)

    def step(self, dlogits: torch.Tensor, hidden: torch.Tensor) -> None:
        self.master.grad = (dlogits.t() @ hidden).float()
        self.opt.step()
        with torch.no_grad():
            self.lm.lm_head.weight.copy_(self.master)


def packed(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


def distill(student, teacher, steps, gen, top=32, temperature=2.0, lr=3e-3):
    head, found = Head(student, lr), []
    cu = packed([97, 160, 33, 128])
    ids = torch.randint(0, student.vocab_size, (cu[-1],), generator=gen, device="cuda")
    with torch.no_grad():
        t = teacher.lm_head(teacher.hidden_states(ids, cu)).float()
        top = min(top, t.shape[1])
        values, places = torch.topk(t, top)
        lse = torch.logsumexp(t / temperature, dim=-1)
    places[torch.tensor(cu[1:], device="cuda") - 1] = -1  # the last token of a sequence predicts nothing
    hidden = student.hidden_states(ids, cu)
    for _ in range(steps):
        loss, _, dlogits = distillation_loss_and_grad(head.logits(hidden), values, places, teacher_lse=lse,
                                                      temperature=temperature)
        head.step(dlogits, hidden)
        found.append(loss)
    return found


def prefer(model, steps, gen, pairs=4, lr=1e-3):
    head, found = Head(model, lr), []
    cu = packed([40 + 7 * (i % 5) for i in range(2 * pairs)])
    ids = torch.randint(0, model.vocab_size, (cu[-1],), generator=gen, device="cuda")
    labels = next_token_labels(ids, cu)
    for s in range(2 * pairs):  # the prompt, the same length in both sequences of a pair, is not trained on
        labels[cu[s]:cu[s] + 10] = -100
    ref = model.score(ids, cu)
    cu_dev = torch.tensor(cu, device="cuda")
    hidden = model.hidden_states(ids, cu)
    for _ in range(steps):
        loss, log_ratios, _, dlogits = preference_loss_and_grad(head.logits(hidden), labels, cu_dev, ref, beta=0.1)
        head.step(dlogits, hidden)
        found.append(loss)
    return found


def reinforce(model, steps, gen, rows=512, lr=3e-3):
    """One sampled token a position; even tokens are rewarded.  Two updates for every sampling."""
    head, found = Head(model, lr), []
    cu = packed([rows // 4] * 4)
    ids = torch.randint(0, model.vocab_size, (cu[-1],), generator=gen, device="cuda")
    hidden = model.hidden_states(ids, cu)
    reference = model.lm_head.weight.detach().clone()
    for _ in range(steps):
        logits = head.logits(hidden)
        actions = torch.multinomial(torch.softmax(logits.float(), -1), 1, generator=gen)[:, 0]
        old = token_logprobs(logits, actions)
        ref = token_logprobs(glue.linear(hidden, reference), actions)
        reward = (actions % 2 == 0).float()
        advantages = (reward - reward.mean()) / (reward.std() + 1e-6)
        for _ in range(2):
            loss, _, _, dlogits = policy_loss_and_grad(head.logits(hidden), actions, old, advantages, ref_logps=ref,
                                                       kl_coef=0.02, entropy_coef=0.001)
            head.step(dlogits, hidden)
        found.append(reward.mean())
    return found


def build(vocab, seed, scale):
    torch.manual_seed(seed)
    lm = KernelDeltaNetLM(vocab_size=vocab, d_model=256, num_layers=3, num_heads=4, d_ff=512, anchor_layers=[1],
                          tie_weights=False)
    with torch.no_grad():
        for p in lm.parameters():
            if p.dim() == 2:
                p.normal_(std=scale / p.shape[1] ** 0.5)
        lm.embed.weight.normal_()
    return lm.to("cuda", torch.bfloat16)


def main(steps=30, vocab=4001, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    teacher, student = build(vocab, seed, 1.5), build(vocab, seed + 1, 1.0)
    out = {"distillation loss": distill(student, teacher, steps, gen), "preference loss": prefer(student, steps, gen),
           "policy reward": reinforce(student, steps, gen)}
    out = {k: [float(x) for x in torch.stack(v).tolist()] for k, v in out.items()}
    for k, v in out.items():
        print(f"{k:18s} first {v[0]:.4f}  last {v[-1]:.4f}  ({len(v)} steps)")
    return out


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--vocab", type=int, default=4001)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args()
    main(a.steps, a.vocab, a.seed)
