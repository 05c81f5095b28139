"""AdamW at the largest array that the C ABI takes, 2^34 elements, bf16
throughout (128 GiB): parts at its ends and across its middle are updated as
the same elements on their own."""
import pytest
import torch

from suika_amd import ShardAdamW

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def test_adamw_of_the_largest_array():
    n, width = 2 ** 34, 10_000
    torch.cuda.empty_cache()
    g = torch.Generator(DEV).manual_seed(1)
    fields = ("param", "exp_avg", "exp_avg_sq")
    state = {"w": {f: torch.zeros(n, dtype=BF16, device=DEV) for f in fields}}
    grad = torch.zeros(n, dtype=BF16, device=DEV)
    parts = [slice(0, width), slice(n // 2 - width // 2, n // 2 + width // 2), slice(n - width, n)]
    small = []
    for p in parts:
        for f in fields:
            state["w"][f][p] = torch.rand(width, generator=g, device=DEV).to(BF16)
        grad[p] = torch.randn(width, generator=g, device=DEV).to(BF16)
        small.append({"w": {f: state["w"][f][p].clone() for f in fields}})
    ShardAdamW(state).step([grad])
    for p, s in zip(parts, small):
        ShardAdamW(s).step([grad[p].clone()])
        assert all(torch.equal(state["w"][f][p], s["w"][f]) for f in fields)
    for at in (width, n // 4, n // 2 + width, n - 2 * width):      # zeros stay zeros
        assert not any(bool(state["w"][f][at:at + 1000].any()) for f in fields)
