"""Sinks of any size under attention_prompt and attention_shared: +inf, or what leaves fp32 in base 2, takes all the weight (zeros),
-inf or as far below has none, NaN is NaN; the same whether a query's keys are one piece or several.  Tolerances: none."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("prefix,own", [(0, 40), (0, 6000), (300, 17), (5000, 600)])
def test_sinks_of_any_size(gpu, prefix, own, dtype):
    from tinygiant_b200 import attention as A
    g, H, KH, hd, dt = torch.Generator(device="cuda").manual_seed(3), 8, 2, 64, getattr(torch, dtype)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dt)  # noqa: E731
    top = torch.finfo(torch.float32).max
    sinks = torch.tensor([math.inf, top, -math.inf, -top, math.nan, 0.5, 3e38, -3e38], device="cuda")
    n = prefix + own
    q, k, v = rand(1, H, hd), rand(KH, n, hd), rand(KH, n, hd)
    cu_q, cu_k = (torch.tensor([0, m], dtype=torch.int32, device="cuda") for m in (1, n))
    prompt = lambda s: A.attention_prompt(q, k.transpose(0, 1), v.transpose(0, 1), cu_q, cu_k, sinks=s)  # noqa: E731
    parts = [x[:, :prefix].contiguous() if prefix else None for x in (k, v)], [x[None, :, prefix:].contiguous() for x in (k, v)]
    lens = torch.tensor([own], dtype=torch.int32, device="cuda")
    shared = lambda s: A.attention_shared(q, *parts[0], *parts[1], lens, sinks=s)  # noqa: E731
    for call in (prompt, shared):
        got, plain, half = call(sinks), call(None), call(torch.full_like(sinks, 0.5))
        assert not bool(got[0, [0, 1, 6]].any()) and torch.equal(got[0, [2, 3, 7]], plain[0, [2, 3, 7]])
        assert bool(torch.isnan(got[0, 4]).all()) and torch.equal(got[0, 5], half[0, 5])
