"""Attention over the paged cache where single tokens, rows or bounds are out of the ordinary. The plain implementation,
the inputs and the tolerances are those of test_paged_gpu.py."""
import pytest
import torch

from test_paged_gpu import _check, _setup

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------- one token above the rest
def _one_loud(n, t, D, kind, size, nats, loud, mean, seed):
    """n rows whose score at token t // 3 lies `nats` above the others'; that token's value is zero, or (loud) zero but
    for one channel `loud` times the others' size."""
    from nano_gpic_b200.ops import paged as P
    kv, table, cu, _, _ = _setup([n], [t], 1, D, 16, kind)
    g = torch.Generator(device="cuda").manual_seed(seed)
    base = torch.randn(D, device="cuda", generator=g)
    q = (base + 0.1 * torch.randn(2 * n, D, device="cuda", generator=g)).view(n, 2 * D).bfloat16()
    k, v = torch.randn(t, D, device="cuda", generator=g), torch.randn(t, D, device="cuda", generator=g) + mean
    z = t // 3
    k[z] = base * (nats * D ** 0.5 / base.square().sum())
    v *= size
    v[z] = 0
    if loud:
        v[z, 5] = size * loud
    P.cache_write(kv, k.bfloat16(), v.bfloat16(), table, torch.zeros(1, dtype=torch.int32, device="cuda"),
                  torch.tensor([0, t], dtype=torch.int32, device="cuda"))
    return q, kv, table, cu


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,t,D", [(1, 2000, 128), (1, 16384, 128), (8, 700, 64), (16, 2000, 128), (32, 3000, 64),
                                   (140, 2000, 128)])
def test_zero_value_of_high_weight(kind, n, t, D):
    """The zero token takes up to 1 - 1e-9 of the probability: the others' part is all of the output and keeps its
    relative precision, whatever their size."""
    for size in (1.0, 0.1, 0.02, 1e-3, 1e-5):
        for nats in (6, 12, 30):
            q, kv, table, cu = _one_loud(n, t, D, kind, size, nats, 0, 1.0, seed=n + D)
            _check(q, kv, table, cu, [n], [t])


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,t,D", [(1, 2000, 128), (8, 700, 64), (32, 3000, 64), (140, 2000, 128)])
def test_one_loud_channel_of_high_weight(kind, n, t, D):
    """That token has one channel of 2^8 to 2^40 times the others' size: the other columns are the others' alone."""
    for size in (1.0, 0.02):
        for loud in (2.0 ** 8, 2.0 ** 20, 2.0 ** 40):
            q, kv, table, cu = _one_loud(n, t, D, kind, size, 12, loud, 0.0, seed=n + D)
            _check(q, kv, table, cu, [n], [t])
