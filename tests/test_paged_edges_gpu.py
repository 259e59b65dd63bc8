"""Attention over the paged cache where single tokens, rows or bounds are out of the ordinary. The plain implementation,
the inputs and the tolerances are those of test_paged_gpu.py."""
import pytest
import torch

from test_paged_gpu import _attn_ref, _check, _fill, _q, _setup

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


# ------------------------------------------------------------------------------------------------------ NaN stays NaN
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n", [1, 8, 200])
@pytest.mark.parametrize("t", [300, 4097, 16385])  # one split; the last key of the longer ones is alone in its split
@pytest.mark.parametrize("where", ["query", "first key", "last key"])
def test_nan_is_not_an_empty_row(kind, n, t, where):
    """A NaN query, or a NaN key that a row sees, makes that row's output and log-sum-exp NaN, split or not; a row that
    saw nothing (o = 0, lse = -inf) is something else, and rows that do not see the NaN keep their results."""
    from nano_gpic_b200.ops import paged as P
    D, H, Hk = 128, 4, 2
    kv, table, cu, _, tot = _setup([n], [t], Hk, D, 16, kind)
    g = torch.Generator(device="cuda").manual_seed(t + n)
    k, v = (torch.randn(t, Hk * D, device="cuda", generator=g).bfloat16() for _ in range(2))
    q = _q(n, H, D)
    if where == "query":
        q[n // 2, D + 3] = float("nan")  # of head 1
    else:
        k[0 if where == "first key" else t - 1, 7] = float("nan")  # of key head 0: heads 0 and 1
    P.cache_write(kv, k, v, table, torch.zeros(1, dtype=torch.int32, device="cuda"),
                  torch.tensor([0, t], dtype=torch.int32, device="cuda"))
    o, lse = P.paged_attn(q, kv, table, tot, cu, n, t)
    ro, rl, A, se = _attn_ref(q, kv, table, [n], [t], D ** -0.5)
    bad = rl.isnan()
    assert int(bad.sum()) == {"query": 1, "first key": 2 * n, "last key": 2}[where]
    o = o.double().view(n, H, D)
    assert torch.equal(lse.isnan(), bad) and torch.equal(o.isnan(), bad[..., None].expand_as(o))
    err, tol = (o - ro).abs(), A * (2 ** -7 + 2 ** -12 + 3 * se[..., None])
    assert (err <= tol)[~bad].all()
    assert ((lse.double() - rl)[~bad].abs() <= (se + 2 ** -19 * (1 + rl.abs()))[~bad]).all()


# -------------------------------------------------------------------------------------------------------- loose bounds
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n", [1, 150])
@pytest.mark.parametrize("bound", [1 << 30, (1 << 31) - 1])
def test_any_length_as_bound(kind, n, bound):
    """max_total far above what the table can hold ("any length"): the same results, from a workspace that goes by the
    table; a sequence that the table cannot hold still sets the status word."""
    from nano_gpic_b200.ops import paged as P
    from nano_gpic_b200.ops import status
    new, total = [n, n, n], [5000, 2100, 170]
    kv, table, cu, _, _ = _setup(new, total, 2, 128, 16, kind)
    _fill(kv, table, total)
    q = _q(3 * n, 16, 128)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    P.paged_attn(q, kv, table, torch.tensor(total, dtype=torch.int32, device="cuda"), cu, n, bound)
    assert torch.cuda.max_memory_allocated() - before < 1 << 28
    _check(q, kv, table, cu, new, total, bound=(n, bound))
    long = torch.tensor([5000, table.shape[1] * 16 + 1, 170], dtype=torch.int32, device="cuda")
    P.paged_attn(q, kv, table, long, cu, n, bound)
    with pytest.raises(RuntimeError, match="page table"):
        status.check()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n", [1, 150])
@pytest.mark.parametrize("bound", [1 << 20, 1 << 29, (1 << 31) - 1])
def test_any_number_of_new_rows_as_bound(kind, n, bound):
    """max_new far above the rows of q: the launch goes by q (eight query heads a key head: rows times heads of such a
    bound pass 2^31), results as with the tight bound of the same kernel."""
    new, total = [n], [400]
    kv, table, cu, _, _ = _setup(new, total, 1, 64, 16, kind)
    _fill(kv, table, total)
    q = _q(n, 8, 64)
    a = _check(q, kv, table, cu, new, total, bound=(n, 400))
    b = _check(q, kv, table, cu, new, total, bound=(bound, 400))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_only_padding_rows(kind):
    """Rows in q that no sequence owns, none at all or max_new = 0: zeros and -inf, as on the CPU, and no error; rows of
    a sequence in spite of max_new = 0 set the status word."""
    from nano_gpic_b200.ops import paged as P
    from nano_gpic_b200.ops import status
    kv, table, cu, pos, tot = _setup([0, 0], [20, 30], 2, 64, 16, kind)
    _fill(kv, table, [20, 30])
    q = _q(5, 4, 64)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    for call in ((q, kv, table, tot, cu, 0, 30), (q, kv, table[:0], tot[:0], none, 3, 30),
                 (q, kv, table[:0], tot[:0], none, 0, 0)):
        o, lse = P.paged_attn(*call)
        status.check()
        assert o.shape == (5, 256) and lse.shape == (5, 4) and (o == 0).all() and (lse == float("-inf")).all()
    P.cache_write(kv, q[:, :128], q[:, :128], table[:0], pos[:0], none)
    k, _ = P.cache_read(kv, table[:0], pos[:0], none, 5)
    assert (k == 0).all()
    P.paged_attn(q, kv, table, tot, torch.tensor([0, 5, 5], dtype=torch.int32, device="cuda"), 0, 30)
    with pytest.raises(RuntimeError, match="bound"):
        status.check()


# ------------------------------------------------------------------------------------------------------------ refusals
def test_scale_pools_of_odd_alignment_are_refused():
    """A contiguous scale pool at an odd place of a byte arena: refused on the host by every call."""
    from nano_gpic_b200.ops import paged as P
    kv, table, cu, pos, tot = _setup([2, 2], [20, 30], 2, 128, 16, "e4m3")
    arena = torch.zeros(2 * kv.k_sf.numel() + 8, dtype=torch.uint8, device="cuda")
    k, q = _q(4, 2, 128), _q(4, 4, 128)
    for at in (1, 2, 3):
        odd = arena[at:at + kv.k_sf.numel()].view(kv.k_sf.shape)
        for sf in ((odd, kv.v_sf), (kv.k_sf, odd)):
            bad = P.PagedKV(kv.k, kv.v, *sf)
            for call in (lambda: P.cache_write(bad, k, k, table, pos, cu), lambda: P.cache_read(bad, table, pos, cu, 4),
                         lambda: P.paged_attn(q, bad, table, tot, cu, 2, 30)):
                with pytest.raises(RuntimeError, match="paged: scale pools"):
                    call()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs a second device")
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_second_device_of_a_process(kind):
    """Both kernels on one device, then on another of the same process: their shared memory is allowed on each."""
    from nano_gpic_b200.ops import paged as P
    for n in (1, 150):
        new, total = [n, n], [200, 180]
        kv, table, cu, _, tot = _setup(new, total, 2, 128, 16, kind)
        _fill(kv, table, total)
        q = _q(2 * n, 4, 128)
        want = P.paged_attn(q, kv, table, tot, cu, n, 200)
        there = [x.to("cuda:1") if x is not None else None for x in (q, table, tot, cu, kv.k, kv.v, kv.k_sf, kv.v_sf)]
        got = P.paged_attn(there[0], P.PagedKV(*there[4:]), *there[1:4], n, 200)
        assert all(torch.equal(x, y.to("cuda:0")) for x, y in zip(want, got))


@pytest.mark.parametrize("scale", [0.0, -0.1, float("nan"), float("inf"), 1e-50, 1e39])
def test_scales_that_are_no_positive_fp32_are_refused(scale):
    from nano_gpic_b200.ops import paged as P
    kv, table, cu, _, tot = _setup([2, 2], [20, 30], 2, 128, 16, "bf16")
    with pytest.raises(RuntimeError, match="paged: scale"):
        P.paged_attn(_q(4, 4, 128), kv, table, tot, cu, 2, 30, scale=scale)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n", [1, 150])
def test_the_least_scale(kind, n):
    """The smallest scales that pass: every visible key weighs the same, masked ones nothing."""
    new, total = [n], [400]
    kv, table, cu, _, _ = _setup(new, total, 2, 128, 16, kind)
    _fill(kv, table, total)
    _check(_q(n, 4, 128), kv, table, cu, new, total, scale=1e-44)
