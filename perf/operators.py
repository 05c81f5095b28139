"""Performance cases of the training-step operators over sharded state.

The state that a plan change moves (parameters, master weights and Adam
moments, with vocabulary-padded embedding and head shards) is trained by
these operators between two changes:

* ``norm``     ``grad_norm``: the 2-norm of all gradients of a share;
* ``clip``     ``clip_grads`` into other tensors (bf16 gradients of the model
               into the f32 ones of an optimizer), norm included;
* ``step``     ``ShardAdamW.step`` with ``max_norm``: norm, clipping and the
               update of every state field, in place;
* ``lookup``   ``vocab_embedding``: rows of a vocabulary shard, scaled;
* ``embed``    the same and ``vocab_embedding_grad``, as a training step runs
               them;
* ``logprob``  ``token_logprobs``: log probabilities of given tokens, entropy
               and, with ``top``, the best alternatives;
* ``loss``     the same and ``token_logprobs_grad``.

State fields (``fields``): ``f32x3`` = f32 param, exp_avg, exp_avg_sq;
``mixed`` = bf16 param with f32 master and moments.  As after a plan change,
a share's tensors lie field by field in one allocation, each at a multiple of
256 bytes and at the same element in every field; the plain forms work on such
a field as a whole, and the fields come back whole.
"""
import math

import torch

own = False

ALIGN = 128          # elements between two tensors' starts in a field: 256 bytes or more
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LR, BETAS, EPS, DECAY = 1e-3, (0.9, 0.95), 1e-8, 0.1
STEPS = 100          # updates that the state has had
MAX_NORM = 1.0
IGNORED = -100       # target of a position that is not scored
GL_STD, GH_STD = 1.0, 0.01


# ------------------------------------------------------------------ cases

def _share(name, op, family, layers, hidden, ffn, vocab, tp, fields="", dtype=""):
    """One rank's share at tensor-parallel degree ``tp``; vocab 0: no embedding."""
    c = {"op": op, "family": family, "layers": layers, "hidden": hidden, "ffn": ffn, "vocab": vocab, "tp": tp}
    if fields:
        c["fields"] = fields
    c["dtype"] = dtype            # of the gradients
    return dict(c, name=name) if name else c


def _embed(name, op, tokens, vocab, shards, at, hidden, dtype, grad="", scale=1.0, pad=0.0, accumulate=False):
    """``vocab`` rows over ``shards`` ranks, of which this is rank ``at``;
    ``pad``: share of the positions that hold one filler token."""
    c = {"op": op, "tokens": tokens, "vocab": vocab, "shards": shards, "at": at, "hidden": hidden, "dtype": dtype,
         "scale": scale, "pad": pad}
    if op == "embed":
        c.update(grad=grad or dtype, accumulate=accumulate)
    return dict(c, name=name) if name else c


def _logits(name, op, rows, columns, vocab, dtype, top=0, masked=0.0):
    """``columns`` logits a row, ``vocab`` of them of real tokens (the others
    pad the head); ``masked``: share of the columns at minus infinity."""
    c = {"op": op, "rows": rows, "columns": columns, "vocab": vocab, "dtype": dtype, "top": top, "masked": masked}
    return dict(c, name=name) if name else c


def listed():
    return [
        # Gradients of one GPT-125M block at TP4, a gradient-accumulation hook's call: launches are all there is.
        _share("norm_gpt125m_block", "norm", "gpt", 1, 768, 3072, 0, 4, dtype="f32"),
        # 8 of Llama2-7B's 32 layers at TP2 with their embedding: bf16 gradients as the backward pass leaves them.
        _share("norm_llama7b", "norm", "llama", 8, 4096, 11008, 32000, 2, dtype="bf16"),
        # GPT-125M whole: bf16 gradients clipped into the optimizer's f32 ones.
        _share("clip_gpt125m", "clip", "gpt", 12, 768, 3072, 50304, 1, dtype="bf16"),
        # The test model's shapes: a step of tensors that hold a few hundred elements each.
        _share("step_gpt_test", "step", "gpt", 2, 16, 64, 128, 2, fields="f32x3", dtype="f32"),
        # The whole GPT-125M share at TP4 in f32: 150 tensors, most of them small.
        _share("step_gpt125m", "step", "gpt", 12, 768, 3072, 50304, 4, fields="f32x3", dtype="f32"),
        # Llama2-7B's share again, mixed precision: the largest state that is stepped here.
        _share("step_llama7b", "step", "llama", 8, 4096, 11008, 32000, 2, fields="mixed", dtype="bf16"),
        # The tokens of one decoding step of 8 sequences, on the second of two vocabulary shards.
        _embed("lookup_decode", "lookup", 8, 32000, 2, 1, 4096, "bf16"),
        # A training batch of 8 x 2048 tokens at Llama2-7B's width, TP2's first vocabulary shard.
        _embed("embed_llama7b", "embed", 16384, 32000, 2, 0, 4096, "bf16"),
        # Ragged sequences at Qwen2-7B's width and vocabulary, TP4, a tenth of the positions padding; the gradient
        # goes to the f32 one that earlier micro-batches filled.
        _embed("embed_qwen7b", "embed", 30011, 152064, 4, 0, 3584, "bf16", grad="f32", scale=59.866518188, pad=0.1,
               accumulate=True),
        # Four sequences decoding with Qwen2-7B's vocabulary under a grammar's mask, 20 alternatives each.
        _logits("logprob_decode", "logprob", 4, 152064, 152064, "bf16", top=20, masked=0.5),
        # The loss of 4 x 2048 positions at Llama2-7B's vocabulary, with its gradient.
        _logits("loss_llama7b", "loss", 8192, 32000, 32000, "bf16"),
        # An odd number of positions, GPT-125M's padded head in f32, 5 alternatives, and the gradient.
        _logits("loss_gpt125m_top", "loss", 2047, 50304, 50257, "f32", top=5),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "clip", "step", "lookup", "embed", "logprob", "loss"])
    if op in ("norm", "clip", "step"):
        while True:
            tp = rng.choice([1, 2, 4, 8])
            hidden = tp * _spread(rng, 3, 4096 // tp)
            fields = rng.choice(["f32x3", "mixed"]) if op == "step" else ""
            dtype = "bf16" if fields == "mixed" or op == "clip" else rng.choice(["f32", "bf16"]) if not fields else "f32"
            c = _share("", op, rng.choice(["gpt", "llama"]), rng.randint(1, 8), hidden, tp * _spread(rng, 5, 11008 // tp),
                       rng.choice([0, _spread(rng, 100, 152064)]), tp, fields=fields, dtype=dtype)
            if _elements(c) < 900e6:
                return c
    if op in ("lookup", "embed"):
        hidden = _spread(rng, 60, 5120)
        tokens = _spread(rng, 1, min(65536, 130_000_000 // hidden))
        shards = rng.choice([1, 2, 4])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        return _embed("", op, tokens, _spread(rng, 300, 152064), shards, rng.randrange(shards), hidden, dtype,
                      grad=rng.choice([dtype, "f32"]), scale=rng.choice([1.0, math.sqrt(hidden)]),
                      pad=rng.choice([0.0, 0.3]), accumulate=rng.choice([False, True]))
    columns = _spread(rng, 300, 152064)
    rows = _spread(rng, 1, min(16384, 250_000_000 // columns))
    vocab = columns - rng.choice([0, 0, rng.randint(1, 127)])
    return _logits("", op, rows, columns, vocab, rng.choice(["bf16", "bf16", "f16", "f32"]),
                   top=rng.choice([0, 1, 5, 20]), masked=rng.choice([0.0, 0.9]))


# ------------------------------------------------------------------ shapes

def _shapes(c):
    """Shapes of a share's tensors: the blocks' and, with a vocabulary, the
    embedding's and the head's rows, cut over the tensor-parallel ranks."""
    H, F, tp, out = c["hidden"], c["ffn"], c["tp"], []
    for _ in range(c["layers"]):
        if c["family"] == "gpt":
            out += [(H,), (H,), (3 * H // tp, H), (3 * H // tp,), (H, H // tp), (H,), (H,), (H,),
                    (F // tp, H), (F // tp,), (H, F // tp), (H,)]
        else:
            out += [(H // tp, H), (H // tp, H), (H // tp, H), (H, H // tp), (F // tp, H), (F // tp, H), (H, F // tp),
                    (H,), (H,)]
    if c["vocab"]:
        out += [(-(-c["vocab"] // tp), H), (-(-c["vocab"] // tp), H), (H,)]
    return out


def _elements(c):
    return sum(math.prod(s) for s in _shapes(c))


def _arena(shapes, dtype):
    """One zeroed allocation and its tensors, each at a multiple of ALIGN elements."""
    at, offsets = 0, []
    for s in shapes:
        offsets.append(at)
        at += -(-math.prod(s) // ALIGN) * ALIGN
    flat = torch.zeros(at, dtype=dtype, device="cuda")
    return flat, [flat[o:o + math.prod(s)].view(s) for o, s in zip(offsets, shapes)]


def _fields(c):
    if c["fields"] == "mixed":
        return {"param": torch.bfloat16, "master": torch.float32, "exp_avg": torch.float32,
                "exp_avg_sq": torch.float32}
    return {"param": torch.float32, "exp_avg": torch.float32, "exp_avg_sq": torch.float32}


# ------------------------------------------------------------------ inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    op = case["op"]

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std)

    if op in ("norm", "clip", "step"):
        shapes = _shapes(case)
        s["grad"], s["grads"] = _arena(shapes, DTYPES[case["dtype"]])
        for i, t in enumerate(s["grads"]):
            t.copy_(normal(*t.shape, std=1e-3 * (1 + i % 7)))
        if op == "clip":
            s["out"], s["outs"] = _arena([(s["grad"].numel(),)], torch.float32)
            s["outs"] = [s["out"][t.storage_offset():t.storage_offset() + t.numel()].view(t.shape) for t in s["grads"]]
        if op == "step":
            tensors = {}
            for f, dt in _fields(case).items():
                s[f], tensors[f] = _arena(shapes, dt)
            for i in range(len(shapes)):
                w = normal(*shapes[i], std=0.02)
                if "master" in tensors:
                    tensors["master"][i].copy_(w)
                tensors["param"][i].copy_(w)
                tensors["exp_avg"][i].copy_(normal(*shapes[i], std=1e-3))
                tensors["exp_avg_sq"][i].copy_(normal(*shapes[i], std=1e-6).abs_())
            s["steps"] = STEPS
            if own:
                import suika_amd
                state = {"p%d" % i: {**{f: tensors[f][i] for f in tensors}, "step": torch.tensor(float(STEPS))}
                         for i in range(len(shapes))}
                s["optimizer"] = suika_amd.ShardAdamW(state, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY)
        return s
    if op in ("lookup", "embed"):
        n, vocab = case["tokens"], case["vocab"]
        rows = -(-vocab // case["shards"])
        u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
        # a token's rank in the vocabulary is spread over its logarithm, as in text
        tokens = (torch.exp(u * math.log(vocab + 1.0)).floor() - 1).clamp(0, vocab - 1).to(torch.int64)
        filler = torch.rand(n, generator=gen, device="cuda") < case["pad"]
        s["tokens"] = torch.where(filler, torch.full_like(tokens, min(3, vocab - 1)), tokens)
        s["start"], s["rows"] = rows * case["at"], rows
        s["weight"] = normal(rows, case["hidden"], std=0.02).to(DTYPES[case["dtype"]])
        if op == "embed":
            s["grad_out"] = normal(n, case["hidden"], std=1e-3).to(DTYPES[case["dtype"]])
            s["grad"] = normal(rows, case["hidden"], std=1e-3).to(DTYPES[case["grad"]]) if case["accumulate"] else None
        return s
    rows, columns, vocab = case["rows"], case["columns"], case["vocab"]
    x = normal(rows, columns, std=2.5)
    if case["masked"]:
        x.masked_fill_(torch.rand(rows, columns, generator=gen, device="cuda") < case["masked"], -math.inf)
    s["logits"] = x.to(DTYPES[case["dtype"]])
    s["targets"] = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    scored = torch.rand(rows, generator=gen, device="cuda") < 0.95
    s["targets"] = torch.where(scored, s["targets"], torch.full_like(s["targets"], IGNORED))
    # a scored token is one that the mask leaves
    s["logits"].scatter_(1, s["targets"].clamp(min=0)[:, None], normal(rows, 1, std=2.5).to(s["logits"].dtype))
    if case["op"] == "loss":
        s["g_logprob"] = normal(rows, std=GL_STD)
        s["g_entropy"] = normal(rows, std=GH_STD)
    return s


# ------------------------------------------------------------------ one pass

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    import suika_amd
    c = s["case"]
    op = c["op"]
    if op == "norm":
        return {"norm": suika_amd.grad_norm(s["grads"])}
    if op == "clip":
        norm = suika_amd.clip_grads(s["grads"], MAX_NORM, out=s["outs"])
        return {"norm": norm, "grad": s["out"]}
    if op == "step":
        norm = s["optimizer"].step(s["grads"], max_norm=MAX_NORM)
        return {"norm": norm, **{f: s[f] for f in _fields(c)}}
    if op in ("lookup", "embed"):
        out = {"out": suika_amd.vocab_embedding(s["tokens"], s["weight"], scale=c["scale"], vocab_start=s["start"])}
        if op == "embed":
            if c["accumulate"]:
                out["grad"] = suika_amd.vocab_embedding_grad(s["tokens"], s["grad_out"], s["rows"], scale=c["scale"],
                                                             vocab_start=s["start"], out=s["grad"], accumulate=True)
            else:
                out["grad"] = suika_amd.vocab_embedding_grad(s["tokens"], s["grad_out"], s["rows"], scale=c["scale"],
                                                             vocab_start=s["start"], dtype=DTYPES[c["grad"]])
        return out
    r = suika_amd.token_logprobs(s["logits"], s["targets"], top=c["top"], vocab=c["vocab"])
    out = {"logprob": r.logprob, "entropy": r.entropy, "lse": r.lse}
    if c["top"]:
        out.update(top_logprob=r.top_logprob, top_index=r.top_index)
    if op == "loss":
        out["grad"] = suika_amd.token_logprobs_grad(s["logits"], s["targets"], r.lse, r.entropy, s["g_logprob"],
                                                    s["g_entropy"], vocab=c["vocab"])
    return out


def _run_plain(s):
    c = s["case"]
    op = c["op"]
    if op in ("norm", "clip", "step"):
        g = s["grad"].float()
        norm = g.square().sum().sqrt()
        if op == "norm":
            return {"norm": norm}
        coef = (MAX_NORM / (norm + 1e-6)).clamp(max=1.0)
        if op == "clip":
            s["out"].copy_(g * coef)
            return {"norm": norm, "grad": s["out"]}
        s["steps"] += 1
        g = g * coef
        p, m, v = s["master" if "master" in s else "param"], s["exp_avg"], s["exp_avg_sq"]
        m.mul_(BETAS[0]).add_(g * (1 - BETAS[0]))
        v.mul_(BETAS[1]).add_(g.square() * (1 - BETAS[1]))
        m_scale = LR / (1 - BETAS[0] ** s["steps"])
        v_scale = math.sqrt(1 - BETAS[1] ** s["steps"])
        p.mul_(1 - LR * DECAY).sub_(m * m_scale / (v.sqrt() / v_scale + EPS))
        if "master" in s:
            s["param"].copy_(p)
        return {"norm": norm, **{f: s[f] for f in _fields(c)}}
    if op in ("lookup", "embed"):
        rows, scale = s["rows"], c["scale"]
        at = s["tokens"] - s["start"]
        inside = (at >= 0) & (at < rows)
        got = s["weight"][at.clamp(0, rows - 1)].float() * scale
        out = {"out": torch.where(inside[:, None], got, 0.0).to(s["weight"].dtype)}
        if op == "embed":
            spare = torch.where(inside, at, rows)          # a row more takes what lies outside
            total = torch.zeros(rows + 1, c["hidden"], device="cuda")
            total.index_add_(0, spare, s["grad_out"].float())
            total = total[:rows] * scale
            if c["accumulate"]:
                out["grad"] = s["grad"].copy_(s["grad"].float() + total)
            else:
                out["grad"] = total.to(DTYPES[c["grad"]])
        return out
    x = s["logits"][:, :c["vocab"]].float()
    target = s["targets"]
    scored = target >= 0
    top = x.max(dim=1, keepdim=True).values
    e = (x - top).exp()
    total = e.sum(dim=1, keepdim=True)
    lse = top + total.log()
    logp = x - lse
    p = e / total
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(dim=1)
    at = target.clamp(min=0)[:, None]
    out = {"logprob": torch.where(scored, logp.gather(1, at)[:, 0], 0.0), "entropy": entropy, "lse": lse[:, 0]}
    if c["top"]:
        best, index = torch.sort(x, dim=1, descending=True, stable=True)
        out.update(top_logprob=best[:, :c["top"]] - lse, top_index=index[:, :c["top"]].contiguous())
    if op == "loss":
        gl = torch.where(scored, s["g_logprob"], 0.0)[:, None]
        grad = torch.zeros(x.shape[0], c["columns"], device="cuda")
        inner = torch.where(p > 0, p * (logp + entropy[:, None]), 0.0)
        grad[:, :c["vocab"]] = -gl * p - s["g_entropy"][:, None] * inner
        grad.scatter_add_(1, at, gl)
        out["grad"] = grad.to(s["logits"].dtype)
    return out


# ------------------------------------------------------------------ what a pass needs

def work(case):
    op = case["op"]
    if op in ("norm", "clip", "step"):
        n, b = _elements(case), DTYPES[case["dtype"]].itemsize
        if op == "norm":
            return {"bytes": n * b, "flops": 2 * n}
        if op == "clip":
            return {"bytes": n * (b + 4), "flops": 3 * n}
        state = sum(dt.itemsize for dt in _fields(case).values())
        reads = state - (2 if case["fields"] == "mixed" else 0)      # a bf16 param is only written
        return {"bytes": n * (b + reads + state), "flops": 18 * n}
    if op in ("lookup", "embed"):
        n, h, b = case["tokens"], case["hidden"], DTYPES[case["dtype"]].itemsize
        rows = -(-case["vocab"] // case["shards"])
        # row r is a token's with probability ln((r+2)/(r+1)) / ln(vocab+1): the tokens of this shard, and the rows they hit
        first = rows * case["at"]
        r = torch.arange(first, max(first, min(case["vocab"], first + rows)), dtype=torch.float64)
        share = (1 - case["pad"]) * torch.log1p(1 / (r + 1)) / math.log(case["vocab"] + 1)
        share += case["pad"] * (r == min(3, case["vocab"] - 1))
        here, hit = n * float(share.sum()), float((1 - (1 - share) ** n).sum())
        moved = 8 * n + b * h * (hit + n)
        if op == "lookup":
            return {"bytes": moved, "flops": h * here}
        # an accumulated gradient changes where a token is; a new one is written whole
        moved += b * h * here + DTYPES[case["grad"]].itemsize * h * (2 * hit if case["accumulate"] else rows)
        return {"bytes": moved, "flops": 2 * h * here}
    n, b = case["rows"] * case["vocab"], DTYPES[case["dtype"]].itemsize
    moved = n * b + case["rows"] * (8 + 12 + 12 * case["top"])
    if op == "logprob":
        return {"bytes": moved, "flops": 6 * n}
    return {"bytes": moved + b * (n + case["rows"] * case["columns"]), "flops": 12 * n}


# ------------------------------------------------------------------ in 64 bits

def _pieces(n, most=1 << 26):
    return [(a, min(n, a + most)) for a in range(0, n, most)]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("norm", "clip", "step"):
        squares = 0.0
        for t in s["grads"]:
            squares += float(torch.linalg.vector_norm(t, dtype=torch.float64)) ** 2
        norm = math.sqrt(squares)
        out = {"norm": torch.tensor(norm, dtype=torch.float64, device="cuda")}
        if op == "norm":
            return out
        coef = min(1.0, MAX_NORM / (norm + 1e-6))
        if op == "clip":
            return {**out, "grad": s["grad"].double() * coef}
        names = list(_fields(case))
        new = {f: torch.zeros(s[f].numel(), dtype=torch.float64, device="cuda") for f in names}
        t = STEPS + 1
        for grad in s["grads"]:
            start = grad.storage_offset()
            for a, b in _pieces(grad.numel()):
                old = {f: s[f][start + a:start + b].double() for f in names}
                g = grad.reshape(-1)[a:b].double() * coef
                avg = old["exp_avg"] + (g - old["exp_avg"]) * (1 - BETAS[0])
                sq = old["exp_avg_sq"] + (g * g - old["exp_avg_sq"]) * (1 - BETAS[1])
                w = old["master" if "master" in old else "param"]
                change = (avg / (1 - BETAS[0] ** t)) / (torch.sqrt(sq / (1 - BETAS[1] ** t)) + EPS)
                w = w - LR * (DECAY * w + change)
                for f, x in (("param", w), ("master", w), ("exp_avg", avg), ("exp_avg_sq", sq)):
                    if f in new:
                        new[f][start + a:start + b] = x
        return {**out, **new}
    if op in ("lookup", "embed"):
        rows, h, scale = s["rows"], case["hidden"], case["scale"]
        table = torch.zeros(rows + 2, h, dtype=torch.float64, device="cuda")     # a row of zeros on either side
        table[1:-1] = s["weight"].double() * scale
        at = (s["tokens"] - s["start"] + 1).clamp(0, rows + 1)
        out = {"out": table.index_select(0, at)}
        if op == "lookup":
            return out
        order = torch.argsort(at, stable=True)
        ends = torch.searchsorted(at[order], torch.arange(rows + 2, device="cuda"), right=True)
        grad = torch.empty(rows, h, dtype=torch.float64, device="cuda")
        for a, b in _pieces(h, max(1, (1 << 28) // case["tokens"])):
            sums = torch.zeros(case["tokens"] + 1, b - a, dtype=torch.float64, device="cuda")
            torch.cumsum(s["grad_out"][order, a:b].double(), dim=0, out=sums[1:])
            grad[:, a:b] = (sums[ends[1:-1]] - sums[ends[:-2]]) * scale
        return {**out, "grad": grad if s["grad"] is None else grad + s["grad"].double()}
    n, vocab, k = case["rows"], case["vocab"], case["top"]
    names = ["logprob", "entropy", "lse"] + (["top_logprob", "top_index"] if k else []) + (["grad"] if op == "loss" else [])
    parts = {f: [] for f in names}
    for a, b in _pieces(n, max(1, (1 << 27) // case["columns"])):
        x = s["logits"][a:b, :vocab].double()
        logp = torch.log_softmax(x, dim=1)
        p = torch.softmax(x, dim=1)
        entropy = torch.special.entr(p).sum(dim=1)
        t = s["targets"][a:b]
        chosen = torch.nn.functional.one_hot(t.clamp(min=0), vocab).bool() & (t >= 0)[:, None]
        parts["logprob"].append(torch.where(chosen, logp, 0.0).sum(dim=1))
        parts["entropy"].append(entropy)
        parts["lse"].append(torch.logsumexp(x, dim=1))
        if k:
            # a key that falls with the logit and, among equal ones, with the column
            order = torch.argsort(-x, dim=1, stable=True)[:, :k]
            parts["top_index"].append(order)
            parts["top_logprob"].append(torch.gather(logp, 1, order))
        if op == "loss":
            gl = torch.where(t >= 0, s["g_logprob"][a:b].double(), 0.0)[:, None]
            spread = torch.where(p > 0, p * (logp + entropy[:, None]), 0.0)
            g = gl * (chosen.double() - p) - s["g_entropy"][a:b].double()[:, None] * spread
            parts["grad"].append(torch.nn.functional.pad(g, (0, case["columns"] - vocab)))
    return {f: torch.cat(v) for f, v in parts.items()}
