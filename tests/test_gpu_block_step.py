"""The operators of a share's matrices together, as a training step uses them:
a gated block between an embedding and a head, its matrices stepped by Muon and
the rest by AdamW, clipped by one norm over both, trained at tensor-parallel
degree 1, resharded to degree 2 and trained on.

The two degrees compute the same numbers in other orders and, on the way, round
partial outputs: every state field after two more steps is compared with that of
training on at degree 1.  A weight moves by at most lr per step where AdamW steps
it, and by lr times an update of singular values up to 1.21 where Muon does; the
degrees' gradients differ by their bf16 roundings, 2^-8 relative a tensor and a
few of them in a row, so updates that are normalised agree to 2^-4 of their size.
"""
import threading

import pytest
import torch

from suika_amd import (VOCAB_PAD, ParamLayout, ShardAdamW, ShardMuon, TensorMeta, counted_names, execute_param_transfer,
                       gated_ffn, grad_square_sum, schedule_param_transfer, split_matrices, token_logprobs, vocab_embedding,
                       vocab_padded)

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
DEV = torch.device("cuda")
VOCAB, HIDDEN, FFN, PAD, LAYERS = 500, 96, 160, 32, 2
LR_MUON, LR_ADAM, MAX_NORM = 0.02, 1e-2, 1.0


def matrices():
    return [f"h.{k}.{n}" for k in range(LAYERS) for n in ("gate", "up", "down")]


def layout(tp):
    rows = vocab_padded(VOCAB, 2, PAD)
    metas = {}
    for r in range(tp):
        m = {"wte": TensorMeta(name="wte", dtype=BF16, shape=(VOCAB, HIDDEN), tp_meta=(0, r, tp), kind=VOCAB_PAD, kind_args=(PAD,)),
             "head": TensorMeta(name="head", dtype=BF16, shape=(rows, HIDDEN), tp_meta=(0, r, tp)),
             "norm": TensorMeta(name="norm", dtype=BF16, shape=(HIDDEN,))}
        for n in matrices():
            down = n.endswith("down")
            m[n] = TensorMeta(name=n, dtype=BF16, shape=(HIDDEN, FFN) if down else (FFN, HIDDEN), tp_meta=(1 if down else 0, r, tp))
        metas[r] = m
    return ParamLayout.from_metas(metas)


def initial_state():
    gen = torch.Generator(DEV).manual_seed(0)
    state = {}
    for name, meta in layout(1).layout[0].items():
        shape = tuple(meta.actual_shape())
        w = torch.ones(shape, device=DEV) if name == "norm" else torch.randn(shape, generator=gen, device=DEV) * 0.1
        if name == "wte":
            w[VOCAB:] = 0
        state[name] = {"param": w.to(BF16), "master": w, "exp_avg": torch.zeros_like(w), "exp_avg_sq": torch.zeros_like(w),
                       "step": torch.tensor(0.0)}
    return state


class Sum(torch.autograd.Function):
    """What the ranks add up; each gets the whole gradient."""
    @staticmethod
    def forward(ctx, *parts):
        ctx.n = len(parts)
        return sum(p.float() for p in parts).to(parts[0].dtype)

    @staticmethod
    def backward(ctx, g):
        return (g.contiguous(),) * ctx.n


def gradients(states, step):
    """Of all ranks, here one after another."""
    tp = len(states)
    gen = torch.Generator(DEV).manual_seed(100 + step)
    tokens = torch.randint(0, VOCAB, (4, 65), generator=gen, device=DEV)
    inputs, targets = tokens[:, :-1].contiguous(), tokens[:, 1:].contiguous()
    params = [{n: e["param"].detach().requires_grad_() for n, e in s.items()} for s in states]
    rows = params[0]["wte"].shape[0]
    x = Sum.apply(*[vocab_embedding(inputs, p["wte"], vocab_start=r * rows) for r, p in enumerate(params)])
    for k in range(LAYERS):
        x = x + Sum.apply(*[gated_ffn(x, p[f"h.{k}.gate"], p[f"h.{k}.up"], p[f"h.{k}.down"]) for p in params])
    x = x * params[0]["norm"]
    logits = torch.cat([x @ p["head"].t() for p in params], dim=-1)
    loss = -token_logprobs(logits, targets, vocab=VOCAB).logprob.mean()
    loss.backward()
    for p in params[1:]:
        p["norm"].grad = params[0]["norm"].grad.clone()
    return [{n: t.grad for n, t in p.items()} for p in params]


def optimizers(states, reduces):
    tp, out = len(states), []
    for r, s in enumerate(states):
        mine = set(matrices())
        muon = ShardMuon({n: s[n] for n in s if n in mine}, lr=LR_MUON, weight_decay=0.01, splits=split_matrices_of(tp, r),
                         all_reduce=reduces[r] if tp > 1 else None)
        out.append((muon, ShardAdamW({n: s[n] for n in s if n not in mine}, lr=LR_ADAM)))
    return out


def split_matrices_of(tp, r):
    cut = split_matrices(layout(tp), r)
    return {n: cut[n] for n in matrices() if n in cut}


def train(states, steps):
    tp = len(states)
    barrier, given = threading.Barrier(tp, timeout=60), [None] * tp

    def reduce_of(r):
        def f(t):
            given[r] = t
            barrier.wait()
            total = sum(x.clone() for x in given)
            torch.cuda.synchronize()
            barrier.wait()
            t.copy_(total)
            torch.cuda.synchronize()
            barrier.wait()
        return f

    opts = optimizers(states, [reduce_of(r) for r in range(tp)])
    plan = layout(tp)
    for k in steps:
        grads = gradients(states, k)
        q = sum(grad_square_sum([grads[r][n] for n in counted_names(plan, r)]) for r in range(tp))
        norms, errors = [None] * tp, []

        def one(r):
            try:
                muon, adam = opts[r]
                norms[r] = muon.step({n: grads[r][n] for n in muon.names}, max_norm=MAX_NORM, square_sum=q)
                again = adam.step({n: grads[r][n] for n in adam.names}, max_norm=MAX_NORM, square_sum=q)
                assert torch.equal(norms[r], again)
            except BaseException as e:
                errors.append(e)
                barrier.abort()

        threads = [threading.Thread(target=one, args=(r,)) for r in range(tp)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        if errors:
            raise errors[0]
        assert all(torch.equal(n, norms[0]) for n in norms)
    return [{**muon.state(), **adam.state()} for muon, adam in opts]


def reshard(states, src, dst):
    ops = schedule_param_transfer(layout(src), layout(dst))
    fields = [(f, "normal") for f in ("param", "master", "exp_avg", "exp_avg_sq")] + [("step", TensorMeta(torch.tensor(0.0, device=DEV)))]
    for s in states:
        for e in s.values():
            e["step"] = e["step"].to(DEV)
    return [execute_param_transfer(ops, {}, DEV, fields, rank=r, fake_source_state_dicts=dict(enumerate(states)))
            for r in range(dst)]


def copies(states):
    return [{n: {f: t.clone() for f, t in e.items()} for n, e in s.items()} for s in states]


def test_step_reshard_step():
    start = train([initial_state()], range(2))
    before = {n: e["master"].clone() for n, e in start[0].items()}
    alone = train(copies(start), range(2, 4))[0]
    halves = reshard(copies(start), 1, 2)
    for n in matrices():
        assert halves[0][n]["master"].numel() * 2 == before[n].numel()
    joined = reshard(train(halves, range(2, 4)), 2, 1)[0]
    for n, e in alone.items():
        rows = VOCAB if n == "wte" else e["master"].shape[0]
        a, b, old = (t[:rows].double() for t in (e["master"], joined[n]["master"], before[n]))
        assert bool((a != old).any()), n
        # two updates each: of their size, the degrees differ by less than 2^-4 a step
        moved = float((a - old).norm())
        assert float((a - b).norm()) <= 2 * 2.0 ** -4 * moved, (n, float((a - b).norm()), moved)
        assert torch.equal(e["param"], e["master"].to(BF16)) and torch.equal(joined[n]["param"], joined[n]["master"].to(BF16))
