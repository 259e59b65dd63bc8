"""Paged key/value cache of a language model: written (bf16, or quantised to e4m3) and read back, and attention of a
chunk of new tokens over it, from one token to long prefills.

A PagedKV is a pool of pages of `page` tokens. A sequence's tokens are found through its row of `table` (int32
[B, pages a sequence]): token t in page table[b, t // page], slot t % page. New tokens are packed: rows cu[b] ..
cu[b + 1] (cu int32 [B + 1]) belong to sequence b. Everything that says where tokens are lives on the device: no call
synchronises, all run on the current stream and can be captured in a graph.

A write and the attention that reads it are ordered by the stream; a pool that is used on several streams needs the
program's own events between them. Slots past a sequence's tokens are never read into a result, whatever they hold (NaN
included). A table entry outside the pool is never followed: it sets the device status word (ops.status), a write or
read skips the token, and the attention rows that would have seen it hold no result.

A key or value that is NaN or infinite belongs to its token: it spreads to every row that sees the token and, a value,
to the rows of the same call whose key tile holds it (probability 0 times NaN), as in any product over tiles.

Scales of an e4m3 pool: one power of two per (token, key head), 2^e with e = ceil(log2(amax / 448)) kept in [-62, 63].
"""
import math

import torch

from .._ext import ext

E4M3_MAX = 448.0
SCALE_LO, SCALE_HI = -62, 63


class PagedKV:
    """Pools k, v [pages, Hk, page, D], bf16 or uint8 (e4m3 bytes, with k_sf, v_sf uint8 [pages, Hk, page] E8M0 scale
    bytes, 4-byte aligned); D is 64 or 128, page a power of two from 8 to 1024. `PagedKV.empty` allocates one."""

    __slots__ = ("k", "v", "k_sf", "v_sf")

    def __init__(self, k, v, k_sf=None, v_sf=None):
        self.k, self.v, self.k_sf, self.v_sf = k, v, k_sf, v_sf

    @classmethod
    def empty(cls, pages, kv_heads, head_dim, page=64, kind="bf16", device="cuda"):
        if kind not in ("bf16", "e4m3"):
            raise ValueError(f"kind must be 'bf16' or 'e4m3', got {kind!r}")
        shape = (pages, kv_heads, page, head_dim)
        dt = torch.bfloat16 if kind == "bf16" else torch.uint8
        k, v = torch.empty(shape, dtype=dt, device=device), torch.empty(shape, dtype=dt, device=device)
        if kind == "bf16":
            return cls(k, v)
        return cls(k, v, *(torch.empty(shape[:3], dtype=torch.uint8, device=device) for _ in range(2)))

    @property
    def page(self):
        return self.k.shape[2]

    def nbytes(self):
        """Bytes of the pools."""
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_sf, self.v_sf) if t is not None)


# ------------------------------------------------------------------------------------------------- CPU restatement
def _check(cache, table, B1, per_seq):
    k, D, page = cache.k, cache.k.shape[3], cache.k.shape[2]
    if D not in (64, 128):
        raise RuntimeError(f"paged: head dim must be 64 or 128, got {D}")
    if page < 8 or page > 1024 or page & (page - 1):
        raise RuntimeError(f"paged: the page size must be a power of two from 8 to 1024, got {page}")
    if (k.dtype == torch.uint8) != (cache.k_sf is not None) or (k.dtype == torch.uint8) != (cache.v_sf is not None):
        raise RuntimeError("paged: e4m3 pools need both scale pools, bf16 pools none")
    if any(t is not None and t.data_ptr() % 4 for t in (cache.k_sf, cache.v_sf)):
        raise RuntimeError("paged: scale pools must be 4-byte aligned")
    if table.dim() != 2 or B1.shape[0] != table.shape[0] + 1 or per_seq.shape[0] != table.shape[0]:
        raise RuntimeError("paged: table [B, n], cu [B + 1] and one length or position per sequence expected")


def _tokens(cache, b, n, table, at):
    """(page, slot) of tokens at .. at + n of sequence b."""
    t = torch.arange(at, at + n)
    return table[b].long()[t // cache.page], t % cache.page


def _quant(x):
    amax = x.abs().amax(-1)
    m, E = torch.frexp(amax / E4M3_MAX)
    e = torch.where(m == 0.5, E - 1, E)
    e = torch.where(amax > 0, e, torch.zeros_like(e)).clamp(SCALE_LO, SCALE_HI)
    q = (x * torch.pow(2.0, -e.float())[..., None]).clamp(-E4M3_MAX, E4M3_MAX)
    return q.to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)


def _dequant(q, sf):
    return q.view(torch.float8_e4m3fn).float() * torch.pow(2.0, sf.float() - 127)[..., None]


def _gather(cache, b, n, table, at):
    """fp32 K and V of tokens at .. at + n of sequence b, [n, Hk, D]."""
    pg, sl = _tokens(cache, b, n, table, at)
    k, v = cache.k[pg, :, sl], cache.v[pg, :, sl]
    if cache.k_sf is not None:
        return _dequant(k, cache.k_sf[pg, :, sl]), _dequant(v, cache.v_sf[pg, :, sl])
    return k.float(), v.float()


# ------------------------------------------------------------------------------------------------------ entry points
def cache_write(cache, k, v, table, pos, cu):
    """Writes the packed rows k, v [T, Hk * D] bf16 (views with a row stride of their own, rows 16-byte aligned) into
    the cache: row r of sequence b becomes token pos[b] + r - cu[b] (pos int32 [B]). Rows past cu[B] are ignored. An
    e4m3 pool takes them quantised, one scale per (token, key head)."""
    if not cache.k.is_cuda:
        _check(cache, table, cu, pos)
        Hk, D = cache.k.shape[1], cache.k.shape[3]
        if k.shape[1] != Hk * D or v.shape != k.shape:
            raise RuntimeError(f"paged: k and v must be [T, {Hk * D}], got {list(k.shape)}, {list(v.shape)}")
        for b in range(table.shape[0]):
            lo, hi = int(cu[b]), min(int(cu[b + 1]), k.shape[0])
            if hi <= lo:
                continue
            pg, sl = _tokens(cache, b, hi - lo, table, int(pos[b]))
            for x, pool, sf in ((k, cache.k, cache.k_sf), (v, cache.v, cache.v_sf)):
                x = x[lo:hi].reshape(hi - lo, Hk, D)
                if sf is None:
                    pool[pg, :, sl] = x
                else:
                    pool[pg, :, sl], sf[pg, :, sl] = _quant(x.float())
        return
    ext().cache_write(cache.k, cache.v, cache.k_sf, cache.v_sf, k, v, table, pos, cu)


def cache_read(cache, table, pos, cu, rows):
    """The inverse of cache_write: packed k, v [rows, Hk * D] bf16, row r of sequence b from token pos[b] + r - cu[b]
    (rows = cu[B], known to the host; rows past cu[B] are zeros). e4m3 values times their scales are exact in bf16."""
    if not cache.k.is_cuda:
        _check(cache, table, cu, pos)
        cols = cache.k.shape[1] * cache.k.shape[3]
        k, v = torch.zeros(rows, cols, dtype=torch.bfloat16), torch.zeros(rows, cols, dtype=torch.bfloat16)
        for b in range(table.shape[0]):
            lo, hi = int(cu[b]), min(int(cu[b + 1]), rows)
            if hi > lo:
                kb, vb = _gather(cache, b, hi - lo, table, int(pos[b]))
                k[lo:hi], v[lo:hi] = kb.reshape(hi - lo, cols), vb.reshape(hi - lo, cols)
        return k, v
    return tuple(ext().cache_read(cache.k, cache.v, cache.k_sf, cache.v_sf, table, pos, cu, rows))


def paged_attn(q, cache, table, total, cu, max_new, max_total, scale=None, causal=True):
    """Attention of the packed new tokens q [T, H * D] bf16 (row stride free) over the cache; H a multiple of the
    cache's key heads (query head h reads key head h // (H / Hk)).

    Sequence b has total[b] tokens in the cache (int32 [B]), its new ones last and already written: row i of its n new
    rows sees tokens 0 .. total[b] - n + i (causal), or all total[b]. A row that sees none gets o = 0, lse = -inf.
    A NaN in a row's query, or in a key that it sees, makes its o and lse NaN.
    max_new and max_total are the host's upper bounds on the new rows and on total of any sequence: they choose the
    launch (as far as q's rows and the table's columns go, so a loose bound is no harm), and a sequence beyond them sets
    the device status word. Rows past cu[B] hold no result. scale (positive) defaults to 1 / sqrt(D).
    Returns (o [T, H * D] bf16, lse [T, H] fp32, natural log)."""
    D = cache.k.shape[3]
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if not q.is_cuda:
        _check(cache, table, cu, total)
        if not 1e-45 <= scale <= 2e38:
            raise RuntimeError("paged: scale must be positive, in fp32's range")
        T, Hk = q.shape[0], cache.k.shape[1]
        H = q.shape[1] // D
        if q.shape[1] % (Hk * D) or H == 0:
            raise RuntimeError(f"paged: q must be [rows, heads * {D}] with a multiple of {Hk} heads, got "
                               f"{list(q.shape)}")
        o, lse = torch.zeros(T, H, D), torch.full((T, H), float("-inf"))
        for b in range(table.shape[0]):
            lo, hi, t = int(cu[b]), min(int(cu[b + 1]), T), int(total[b])
            if hi <= lo or t <= 0:
                continue
            kb, vb = (x.repeat_interleave(H // Hk, 1) for x in _gather(cache, b, t, table, 0))
            s = torch.einsum("ihd,jhd->hij", q[lo:hi].float().view(hi - lo, H, D), kb) * scale
            if causal:
                see = torch.arange(t)[None] <= torch.arange(t - (hi - lo), t)[:, None]
                s = s.masked_fill(~see, float("-inf"))
            z = torch.logsumexp(s, -1)
            p = torch.exp(s - torch.where(z.isinf(), 0.0, z)[..., None])
            o[lo:hi], lse[lo:hi] = torch.einsum("hij,jhd->ihd", p, vb), z.t()
        return o.reshape(T, H * D).to(torch.bfloat16), lse
    return tuple(ext().paged_attn(q, cache.k, cache.v, cache.k_sf, cache.v_sf, table, total, cu, max_new, max_total,
                                  scale, causal))
