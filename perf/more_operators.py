"""Performance cases of the operators on a share's matrices.

Most of the state that a plan change moves are the blocks' matrices, cut over
the tensor-parallel ranks.  These are the products that train them:

* ``ffn``    ``gated_ffn``: the gated feed-forward block of a shard, forward;
* ``train``  the same, keeping its projections, and ``gated_ffn_grad``: the
             gradients of the input and of all three matrices;
* ``ortho``  ``orthogonalize``: Newton-Schulz products over a list of matrices;
* ``muon``   ``ShardMuon.step``: momentum, orthogonalised update, decay and the
             rounding of the parameters, in place.

State fields (``fields``): ``f32`` = f32 param and exp_avg, f32 gradients;
``mixed`` = bf16 param with f32 master and exp_avg, bf16 gradients.  A share's
tensors lie field by field in one allocation, each at a multiple of 256 bytes
and at the same element in every field, and the fields come back whole.
"""
import math

import torch

own = False

ALIGN = 128          # elements between two tensors' starts in a field: 256 bytes or more
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
LR, MOMENTUM, DECAY, RMS = 1e-3, 0.95, 0.1, 0.2


# ------------------------------------------------------------------ cases

def _ffn(name, op, tokens, hidden, ffn, dtype, activation="silu"):
    """``ffn`` columns of the block are this rank's."""
    c = {"op": op, "tokens": tokens, "hidden": hidden, "ffn": ffn, "dtype": dtype, "activation": activation}
    return dict(c, name=name) if name else c


def _share(name, op, layers, hidden, q, kv, ffn, gated=True, dtype="", fields=""):
    """The matrices of ``layers`` blocks: this rank's rows of the query, key
    and value projections (fused where the block is not gated) and columns of
    the output projection, and its part of the feed-forward block."""
    c = {"op": op, "layers": layers, "hidden": hidden, "q": q, "kv": kv, "ffn": ffn, "gated": gated}
    if op == "ortho":
        c["dtype"] = dtype
    else:
        c["fields"] = fields
    return dict(c, name=name) if name else c


def listed():
    return [
        # One sequence decoding on a Qwen2-7B shard at TP4: the weights' bytes are all there is.
        _ffn("ffn_decode_qwen7b", "ffn", 1, 3584, 4736, "bf16"),
        # 24 sequences decoding on a Llama2-7B shard at TP2.
        _ffn("ffn_decode_llama7b", "ffn", 24, 4096, 5504, "bf16"),
        # An odd number of prompt tokens scored on a Llama2-13B shard at TP4, in f16.
        _ffn("ffn_score_llama13b", "ffn", 2047, 5120, 3456, "f16"),
        # A short ragged batch of a small f32 model with GELU gates, trained.
        _ffn("train_small_f32", "train", 509, 768, 2050, "f32", "gelu"),
        # A fine-tuning batch of 1021 tokens, Qwen2-7B at TP4.
        _ffn("train_qwen7b", "train", 1021, 3584, 4736, "bf16"),
        # A training batch of 4 x 2048 tokens, Llama2-7B at TP2.
        _ffn("train_llama7b", "train", 8192, 4096, 5504, "bf16"),
        # The test model's matrices: a few hundred elements each, launches are all there is.
        _share("ortho_gpt_test", "ortho", 2, 16, 8, 8, 32, gated=False, dtype="f32"),
        # GPT-125M's share at TP4 in f32: 48 matrices of 192 to 768 rows.
        _share("ortho_gpt125m", "ortho", 12, 768, 192, 192, 768, gated=False, dtype="f32"),
        # One block of Llama2-7B at TP2, bf16 momentum in, bf16 update out.
        _share("ortho_llama7b", "ortho", 1, 4096, 2048, 2048, 5504, dtype="bf16"),
        # The test model stepped.
        _share("muon_llama_test", "muon", 2, 16, 8, 8, 32, fields="f32"),
        # Two blocks of Qwen2-7B at TP4: one key and value head of 128 rows beside the wide matrices.
        _share("muon_qwen7b", "muon", 2, 3584, 896, 128, 4736, fields="mixed"),
        # Two blocks of Llama2-7B at TP2, mixed precision: the largest state that is stepped here.
        _share("muon_llama7b", "muon", 2, 4096, 2048, 2048, 5504, fields="mixed"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["ffn", "train", "train", "ortho", "muon"])
    if op in ("ffn", "train"):
        while True:
            unit = rng.choice([1, 2, 8, 64])
            hidden, ffn = unit * _spread(rng, 3 + 16 // unit, 5120 // unit), unit * _spread(rng, 3 + 16 // unit, 11008 // unit)
            tokens = _spread(rng, 1, 8192)
            dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
            if tokens * hidden * ffn * (8 if dtype == "f32" else 1) <= 8192 * 4096 * 5504:
                return _ffn("", op, tokens, hidden, ffn, dtype, rng.choice(["silu", "silu", "gelu", "gelu_tanh"]))
    largest = work(listed()[-1])["flops"]
    while True:
        unit = rng.choice([1, 4, 16, 64])
        hidden = unit * _spread(rng, 2 + 8 // unit, 4096 // unit)
        q = max(1, hidden // rng.choice([1, 2, 4, 8]))
        kv = max(1, q // rng.choice([1, 1, 4, 7]))
        c = _share("", op, rng.randint(1, 8), hidden, q, kv, unit * _spread(rng, 2 + 8 // unit, 5504 // unit),
                   gated=rng.random() < 0.5, dtype=rng.choice(["f32", "bf16", "f16"]), fields=rng.choice(["f32", "mixed"]))
        if work(c)["flops"] <= largest:
            return c


# ------------------------------------------------------------------ shapes

def _shapes(c):
    """Shapes of a share's matrices."""
    H, q, kv, F = c["hidden"], c["q"], c["kv"], c["ffn"]
    if c["gated"]:
        return c["layers"] * [(q, H), (kv, H), (kv, H), (H, q), (F, H), (F, H), (H, F)]
    return c["layers"] * [(q + 2 * kv, H), (H, q), (F, H), (H, F)]


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
        return {"param": torch.bfloat16, "master": torch.float32, "exp_avg": torch.float32}
    return {"param": torch.float32, "exp_avg": torch.float32}


# ------------------------------------------------------------------ inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std)

    if case["op"] in ("ffn", "train"):
        T, H, F, dtype = case["tokens"], case["hidden"], case["ffn"], DTYPES[case["dtype"]]
        s["x"] = normal(T, H).to(dtype)                       # as a norm leaves it
        s["gate"] = normal(F, H, std=H ** -0.5).to(dtype)
        s["up"] = normal(F, H, std=H ** -0.5).to(dtype)
        s["down"] = normal(H, F, std=F ** -0.5).to(dtype)
        if case["op"] == "train":
            s["grad_out"] = normal(T, H, std=1e-2).to(dtype)
        return s
    shapes = _shapes(case)
    dtype = DTYPES[case["dtype"]] if case["op"] == "ortho" else DTYPES["bf16" if case["fields"] == "mixed" else "f32"]
    s["grad"], s["grads"] = _arena(shapes, dtype)
    for i, t in enumerate(s["grads"]):
        # a few directions of a gradient are much larger than the rest
        rank = max(1, min(t.shape) // 16)
        low = normal(t.shape[0], rank) @ normal(rank, t.shape[1])
        t.copy_((low + normal(*t.shape)).mul_(1e-4 * (1 + i % 7)))
    if case["op"] == "muon":
        tensors = {}
        for f, dt in _fields(case).items():
            s[f], tensors[f] = _arena(shapes, dt)
        for i, shape in enumerate(shapes):
            w = normal(*shape, std=0.02)
            if "master" in tensors:
                tensors["master"][i].copy_(w)
            tensors["param"][i].copy_(w)
            tensors["exp_avg"][i].copy_(normal(*shape, std=1e-4))
        s["tensors"] = tensors
        if own:
            import suika_amd
            state = {"p%d" % i: {f: tensors[f][i] for f in tensors} for i in range(len(shapes))}
            s["optimizer"] = suika_amd.ShardMuon(state, lr=LR, momentum=MOMENTUM, weight_decay=DECAY, ns_steps=STEPS,
                                                 ns_coefficients=COEFFICIENTS, eps=EPS, adjust_lr="match_rms_adamw")
    return s


# ------------------------------------------------------------------ one pass

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    import suika_amd
    c = s["case"]
    if c["op"] == "ffn":
        return {"out": suika_amd.gated_ffn(s["x"], s["gate"], s["up"], s["down"], activation=c["activation"])}
    if c["op"] == "train":
        r = suika_amd.gated_ffn(s["x"], s["gate"], s["up"], s["down"], activation=c["activation"], keep=True)
        grads = suika_amd.gated_ffn_grad(s["x"], s["gate"], s["up"], s["down"], r.gate, r.up, s["grad_out"],
                                         activation=c["activation"])
        return {"out": r.out, "x": grads[0], "gate": grads[1], "up": grads[2], "down": grads[3]}
    if c["op"] == "ortho":
        return suika_amd.orthogonalize(s["grads"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
    s["optimizer"].step(s["grads"])
    return {f: s[f] for f in _fields(c)}


def _act(a, activation):
    """The activation and its derivative."""
    if activation == "gelu":
        phi = 0.5 * (1 + torch.erf(a * math.sqrt(0.5)))
        return a * phi, phi + a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)
    if activation == "silu":
        p = 1 / (1 + torch.exp(-a))
        return a * p, p * (1 + a * (1 - p))
    t = torch.tanh(math.sqrt(2 / math.pi) * (a + 0.044715 * a * a * a))
    slope = math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * a * a)
    return 0.5 * a * (1 + t), 0.5 * (1 + t) + 0.5 * a * (1 - t * t) * slope


def _orthogonal(g):
    """Newton-Schulz products, the shorter side's Gram matrix first."""
    x = g / g.square().sum().sqrt().clamp(min=EPS)
    wide = x.shape[0] <= x.shape[1]
    if not wide:
        x = x.t()
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        gram = x @ x.t()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x if wide else x.t()


def _run_plain(s):
    c = s["case"]
    if c["op"] in ("ffn", "train"):
        dtype = s["x"].dtype
        x, gate, up, down = (s[k].float() for k in ("x", "gate", "up", "down"))
        a, b = x @ gate.t(), x @ up.t()
        f, slope = _act(a, c["activation"])
        h = f * b
        out = {"out": (h @ down.t()).to(dtype)}
        if c["op"] == "train":
            dy = s["grad_out"].float()
            dh = dy @ down
            da, db = dh * b * slope, dh * f
            out.update(x=(da @ gate + db @ up).to(dtype), gate=(da.t() @ x).to(dtype), up=(db.t() @ x).to(dtype),
                       down=(dy.t() @ h).to(dtype))
        return out
    if c["op"] == "ortho":
        return [_orthogonal(g.float()).to(g.dtype) for g in s["grads"]]
    t = s["tensors"]
    weights = t["master" if "master" in t else "param"]
    for i, g in enumerate(s["grads"]):
        g = g.float() * (1 - MOMENTUM)
        m = t["exp_avg"][i].mul_(MOMENTUM).add_(g)
        update = _orthogonal(m * MOMENTUM + g)
        weights[i].mul_(1 - LR * DECAY).sub_(update * (LR * RMS * math.sqrt(max(g.shape))))
        if "master" in t:
            t["param"][i].copy_(weights[i])
    return {f: s[f] for f in _fields(c)}


# ------------------------------------------------------------------ what a pass needs

def work(case):
    if case["op"] in ("ffn", "train"):
        T, H, F, b = case["tokens"], case["hidden"], case["ffn"], DTYPES[case["dtype"]].itemsize
        if case["op"] == "ffn":
            return {"bytes": b * (2 * T * H + 3 * H * F), "flops": 6 * T * H * F}
        return {"bytes": b * (4 * T * H + 6 * H * F), "flops": 18 * T * H * F}
    flops = elements = 0
    for r, k in _shapes(case):
        m, n = min(r, k), max(r, k)
        # the Gram matrix and its square are symmetric: half of their products
        flops += STEPS * (m * m * n + m * m * m + 2 * m * m * n)
        elements += m * n
    if case["op"] == "ortho":
        return {"bytes": 2 * elements * DTYPES[case["dtype"]].itemsize, "flops": flops}
    # gradient in, weight and momentum in and out, a copy of the weight out
    return {"bytes": elements * (2 + 8 + 8 + 2 if case["fields"] == "mixed" else 4 + 8 + 8), "flops": flops}


# ------------------------------------------------------------------ in 64 bits

def _orthogonal_exact(g):
    """The same polynomial from the other side, on whole powers: with
    S = X^T X of the shorter side, X <- X (a I + b S + c S S)."""
    x = g / torch.clamp(torch.linalg.vector_norm(g), min=EPS)
    flip = x.shape[1] > x.shape[0]
    x = x.t().contiguous() if flip else x
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        s = torch.mm(x.t().contiguous(), x)
        p = torch.mm(s, s).mul_(c).add_(s, alpha=b)
        p.diagonal().add_(a)
        x = torch.mm(x, p)
    return x.t() if flip else x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("ffn", "train"):
        leaves = [s[k].double().requires_grad_(case["op"] == "train") for k in ("x", "gate", "up", "down")]
        x, gate, up, down = leaves
        a = torch.nn.functional.linear(x, gate)
        act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
               "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[case["activation"]]
        y = torch.nn.functional.linear(act(a) * torch.nn.functional.linear(x, up), down)
        if case["op"] == "ffn":
            return {"out": y}
        grads = torch.autograd.grad(y, leaves, s["grad_out"].double())
        return {"out": y.detach(), "x": grads[0], "gate": grads[1], "up": grads[2], "down": grads[3]}
    if case["op"] == "ortho":
        return [_orthogonal_exact(g.double()) for g in s["grads"]]
    out = {f: torch.zeros(s[f].numel(), dtype=torch.float64, device="cuda") for f in _fields(case)}
    t = s["tensors"]
    for i, g in enumerate(s["grads"]):
        at = slice(g.storage_offset(), g.storage_offset() + g.numel())
        m, g = t["exp_avg"][i].double(), g.double()
        m = m + (1 - MOMENTUM) * (g - m)
        u = g + MOMENTUM * (m - g)
        w = t["master" if "master" in t else "param"][i].double()
        w = w - LR * (DECAY * w + RMS * math.sqrt(max(w.shape)) * _orthogonal_exact(u))
        out["exp_avg"][at] = m.reshape(-1)
        out["param"][at] = w.reshape(-1)
        if "master" in out:
            out["master"][at] = w.reshape(-1)
    return out
