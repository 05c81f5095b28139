"""Which rank counts which gradient in a global norm: every element once,
whatever degrees the replicas of a parameter have.  The counted shards' sums of
squares add up to that of the whole gradients."""
import pytest
import torch

from suika_amd import QKV_HEADS, VOCAB_PAD, ParamLayout, TensorMeta, counted_names

F32 = torch.float32
VOCAB, PAD = 21, 4
QKV = (8, 4, 2)      # query heads, key heads, rows of a head
SHAPES = {"w": (8, 3), "row": (3, 8), "wte": (VOCAB, 3), "qkv": ((8 + 2 * 4) * 2, 3), "norm": (5,)}


def metas(index, deg):
    tp = None if deg == 1 else (0, index, deg)
    return {
        "w": TensorMeta(name="w", dtype=F32, shape=SHAPES["w"], tp_meta=tp),
        "row": TensorMeta(name="row", dtype=F32, shape=SHAPES["row"], tp_meta=(1, index, deg)),
        "wte": TensorMeta(name="wte", dtype=F32, shape=SHAPES["wte"], tp_meta=(0, index, deg), kind=VOCAB_PAD,
                          kind_args=(PAD,)),
        "qkv": TensorMeta(name="qkv", dtype=F32, shape=SHAPES["qkv"], tp_meta=(0, index, deg), kind=QKV_HEADS,
                          kind_args=QKV),
        "norm": TensorMeta(name="norm", dtype=F32, shape=SHAPES["norm"]),
    }


def shard(meta, whole):
    if not meta.is_tp():
        return whole
    dim, index, deg = meta.tp_meta
    if meta.kind == VOCAB_PAD:
        whole = torch.nn.functional.pad(whole, (0, 0, 0, meta.padded_rows() - len(whole)))
    if meta.kind == QKV_HEADS:
        n_q, n_kv, d = QKV
        return torch.cat([p.chunk(deg)[index] for p in whole.split([n_q * d, n_kv * d, n_kv * d])])
    return whole.chunk(deg, dim)[index]


@pytest.mark.parametrize("order", ["groups", "reversed"])
@pytest.mark.parametrize("degrees", [(1,), (2,), (2, 2), (2, 1), (1, 2), (2, 2, 1), (1, 2, 2), (1, 1, 2), (4, 2, 1),
                                     (1, 4, 2), (2, 4), (4, 4, 2)])
def test_every_element_counts_once(degrees, order):
    shards = [(i, d) for d in degrees for i in range(d)]
    if order == "reversed":
        shards.reverse()
    layout = ParamLayout.from_metas({r: metas(i, d) for r, (i, d) in enumerate(shards)})
    gen = torch.Generator().manual_seed(0)
    # whole numbers: the sums of squares are exact in any order
    whole = {n: torch.randint(-9, 10, s, generator=gen).double() for n, s in SHAPES.items()}
    for n, g in whole.items():
        total = sum(float(shard(layout.layout[r][n], g).square().sum())
                    for r in layout.layout if n in counted_names(layout, r))
        assert total == float(g.square().sum()), n


def test_a_degree_whose_shards_are_not_all_there_does_not_count():
    one = TensorMeta(name="w", dtype=F32, shape=(4, 4), tp_meta=(0, 0, 2))
    whole = TensorMeta(name="w", dtype=F32, shape=(4, 4))
    layout = ParamLayout.from_metas({0: {"w": one}, 1: {"w": whole}, 2: {"w": whole}})
    assert [counted_names(layout, r) for r in range(3)] == [[], ["w"], []]


def test_parameters_of_other_stages():
    w, v = TensorMeta(name="w", dtype=F32, shape=(4,)), TensorMeta(name="v", dtype=F32, shape=(4,))
    layout = ParamLayout.from_metas({3: {"w": w}, 1: {"v": v}, 7: {"v": v, "w": w}})
    assert [counted_names(layout, r) for r in (1, 3, 7)] == [["v"], ["w"], []]
