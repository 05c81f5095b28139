"""Train, change the plan, train on: the operators of a training step on the
state that a plan change moves.

A small language model -- a vocabulary-padded embedding, one linear layer and a
head -- is trained on synthetic text at tensor-parallel degree 1.  Its state
(bf16 param, f32 master and Adam moments) is then resharded to degree 2 and
trained on as two ranks' shards, here both on one GPU:

* ``vocab_embedding``   each rank's rows of the tokens, which add up;
* ``token_logprobs``    the loss, from the gathered logits, with the entropy
                        and the best alternatives of the last position;
* ``grad_square_sum``   over the gradients that each rank counts
                        (``counted_names``), added up over the ranks;
* ``ShardAdamW.step``   clipping by that sum and the update, rank by rank.

    python examples/train_and_reshard.py [--steps 30]

prints the loss of every fifth step, before and after the change, next to the
loss of the same steps without one.
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from suika_amd import (VOCAB_PAD, ParamLayout, ShardAdamW, TensorMeta, counted_names, execute_param_transfer,  # noqa: E402
                       grad_square_sum, schedule_param_transfer, token_logprobs, vocab_embedding, vocab_padded)

VOCAB, HIDDEN, PAD = 1000, 128, 64
BATCH, LENGTH = 8, 64
FIELDS = ("param", "master", "exp_avg", "exp_avg_sq")
MAX_NORM = 1.0


def layout(tp):
    """The model's layout: the embedding's rows padded and cut, the linear
    layer and the head column parallel, the head's rows padded to the same."""
    rows = vocab_padded(VOCAB, 2, PAD)         # the head's, whatever the degree
    bf16, metas = torch.bfloat16, {}
    for r in range(tp):
        metas[r] = {
            "wte.weight": TensorMeta(name="wte.weight", dtype=bf16, shape=(VOCAB, HIDDEN), tp_meta=(0, r, tp),
                                     kind=VOCAB_PAD, kind_args=(PAD,)),
            "proj.weight": TensorMeta(name="proj.weight", dtype=bf16, shape=(HIDDEN, HIDDEN), tp_meta=(0, r, tp)),
            "norm.weight": TensorMeta(name="norm.weight", dtype=bf16, shape=(HIDDEN,)),
            "head.weight": TensorMeta(name="head.weight", dtype=bf16, shape=(rows, HIDDEN), tp_meta=(0, r, tp)),
        }
    return ParamLayout.from_metas(metas)


def initial_state(device, seed=0):
    gen = torch.Generator(device=device).manual_seed(seed)
    state = {}
    for name, meta in layout(1).layout[0].items():
        shape = tuple(meta.actual_shape())
        if name == "norm.weight":
            w = torch.ones(shape, device=device)
        else:
            w = torch.randn(shape, generator=gen, device=device) * 0.05
        if name == "wte.weight":
            w[VOCAB:] = 0
        state[name] = {"param": w.to(torch.bfloat16), "master": w, "exp_avg": torch.zeros_like(w),
                       "exp_avg_sq": torch.zeros_like(w), "step": torch.tensor(0.0)}
    return state


def text(device, step):
    """Tokens that follow from their predecessors, mostly."""
    gen = torch.Generator(device=device).manual_seed(1000 + step)
    first = torch.randint(0, VOCAB, (BATCH, 1), generator=gen, device=device)
    tokens = (first * 7 + 31 * torch.arange(LENGTH + 1, device=device)) % VOCAB
    noise = torch.rand(BATCH, LENGTH + 1, generator=gen, device=device) < 0.1
    return torch.where(noise, torch.randint(0, VOCAB, tokens.shape, generator=gen, device=device), tokens)


def train_step(states, optimizers, plan, tokens):
    """One step of all ranks; the loss, the gradients' norm and the
    alternatives at the last position."""
    tp = len(states)
    params = [{n: e["param"].detach().requires_grad_() for n, e in s.items()} for s in states]
    inputs, targets = tokens[:, :-1].contiguous(), tokens[:, 1:].contiguous()
    rows = params[0]["wte.weight"].shape[0]
    # the ranks' rows add up (an all-reduce), and so do the layers' columns side by side (all-gathers)
    x = sum(vocab_embedding(inputs, p["wte.weight"], vocab_start=r * rows).float() for r, p in enumerate(params))
    x = x.to(torch.bfloat16)
    h = torch.cat([x @ p["proj.weight"].t() for p in params], dim=-1)
    x = x + torch.nn.functional.silu(h) * params[0]["norm.weight"]
    logits = torch.cat([x @ p["head.weight"].t() for p in params], dim=-1)
    scores = token_logprobs(logits, targets, top=3, vocab=VOCAB)
    loss = -scores.logprob.mean()
    loss.backward()
    # a replicated parameter's gradient is the same on every rank
    for p in params[1:]:
        p["norm.weight"].grad = params[0]["norm.weight"].grad.clone()
    grads = [{n: t.grad for n, t in p.items()} for p in params]
    square_sum = sum(grad_square_sum([grads[r][n] for n in counted_names(plan, r)]) for r in range(tp))
    for r in range(tp):
        norm = optimizers[r].step(grads[r], max_norm=MAX_NORM, square_sum=square_sum)
    return loss.detach(), norm, scores.top_index[:, -1]


def optimizers_of(states):
    return [ShardAdamW(s, lr=1e-2, betas=(0.9, 0.95), weight_decay=0.01) for s in states]


def reshard(states, src_tp, dst_tp, device):
    """The ranks' states at degree ``src_tp`` as those at ``dst_tp``."""
    ops = schedule_param_transfer(layout(src_tp), layout(dst_tp))
    step = TensorMeta(states[0]["wte.weight"]["step"])
    fields = [(f, "normal") for f in FIELDS] + [("step", step)]
    out = []
    for r in range(dst_tp):
        out.append(execute_param_transfer(ops, {}, device, fields, rank=r,
                                          fake_source_state_dicts=dict(enumerate(states))))
    return out


def run(steps=30, device="cuda", change_at=None):
    """Losses of ``steps`` steps; from step ``change_at`` on at degree 2."""
    device = torch.device(device)
    states, tp = [initial_state(device)], 1
    optimizers, losses = optimizers_of(states), []
    for k in range(steps):
        if k == change_at:
            states = reshard([o.state() for o in optimizers], 1, 2, device)
            optimizers, tp = optimizers_of(states), 2
        loss, norm, best = train_step(states, optimizers, layout(tp), text(device, k))
        losses.append(loss)
    return [float(x) for x in losses]


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=30)
    a = ap.parse_args()
    alone = run(a.steps)
    changed = run(a.steps, change_at=a.steps // 2)
    for k in range(0, a.steps, 5):
        where = "TP2" if k >= a.steps // 2 else "TP1"
        print(f"step {k:3d}  {where}  loss {changed[k]:.4f}  without the change {alone[k]:.4f}")


if __name__ == "__main__":
    main()
