"""The caption language model (Qwen3 architecture) on the framework's kernels: the frozen encoder of
Qwen3TextEncoder without a foreign eager model, over a paged key/value cache.

A block is  h, s = add_rms(delta, s);  q, k, v = h Wqkv;  q, k per-head RMSNorm + RoPE;  cache_write;  paged_attn;
delta = o Wo;  h, s = add_rms(delta, s);  delta = (silu(h Wg) * (h Wu)) Wd.  The residual stream stays bf16, every norm
takes the addition in front of it, and with fp8="mx" the norms hand their output to the projections in MXFP8.

`TextLM.encode` takes a padded batch as the conditioner does; `TextLM.extend` appends packed new tokens (whole prompts,
chunks of them, or one token each) to the sequences of a `TextCache`.
"""
import torch

from ..ops import gemm as G
from ..ops import mx as MXO
from ..ops import norm as N
from ..ops import paged as P

BF16 = torch.bfloat16


class TextCache:
    """One PagedKV per layer and the page table they share, for `seqs` sequences of at most `max_tokens` tokens."""

    def __init__(self, lm, seqs, max_tokens, kind="bf16", page=64):
        self.page, self.max_tokens = page, max_tokens
        per = (max_tokens + page - 1) // page
        self.table = torch.arange(seqs * per, dtype=torch.int32, device=lm.device).view(seqs, per)
        self.layers = [P.PagedKV.empty(max(1, seqs * per), lm.kv_heads, lm.head_dim, page, kind, lm.device)
                       for _ in lm.blocks]
        self.lens = [0] * seqs  # tokens of each sequence so far


WEIGHTS = tuple(f"{n}.weight" for n in (
    "embed_tokens", "input_layernorm", "post_attention_layernorm", "q_norm", "k_norm", "q_proj", "k_proj", "v_proj",
    "o_proj", "gate_proj", "up_proj", "down_proj", "norm"))
# rotary tables that are fixed frequencies and nothing else
ROPE_TYPES = ("default", "linear", "llama3")


def check_model(model):
    """Raises for what a Qwen3Model may have and the blocks above do not compute."""
    c = model.config
    # (configs without layer_types say it once for all layers)
    kinds = getattr(c, "layer_types", None) or [
        "sliding_attention" if getattr(c, "use_sliding_window", False) else "full_attention"]
    if set(kinds) != {"full_attention"}:
        raise ValueError("TextLM: full attention in every layer expected, the model has a sliding window")
    if c.hidden_act not in ("silu", "swish"):
        raise ValueError(f"TextLM: hidden_act must be 'silu', got {c.hidden_act!r}")
    rope = getattr(c, "rope_parameters", None) or getattr(c, "rope_scaling", None) or {}
    kind = rope.get("rope_type", rope.get("type", "default"))
    if kind not in ROPE_TYPES or getattr(model.rotary_emb, "attention_scaling", 1.0) != 1.0:
        raise ValueError(f"TextLM: rotary embedding of type {ROPE_TYPES} without attention scaling expected, got "
                         f"{kind!r}")
    rest = sorted(k for k in model.state_dict() if not k.startswith("rotary_emb.") and not k.endswith(WEIGHTS))
    if rest:
        raise ValueError(f"TextLM: no use for the model's {rest}")


class TextLM:
    """Weights of a transformers Qwen3Model, laid out for the kernels. A model with anything these blocks do not compute
    (biases, a sliding window, another activation, a scaled or length-dependent rotary embedding) is refused."""

    def __init__(self, model, fp8=None):
        if fp8 not in (None, "mx"):
            raise ValueError(f"fp8 must be None or 'mx', got {fp8!r}")
        check_model(model)
        c = model.config
        self.fp8 = fp8
        self.heads, self.kv_heads = c.num_attention_heads, c.num_key_value_heads
        self.head_dim = getattr(c, "head_dim", None) or c.hidden_size // c.num_attention_heads
        self.eps = c.rms_norm_eps
        sd = {k: v.detach() for k, v in model.state_dict().items()}
        self.device = sd["embed_tokens.weight"].device
        self.embed = sd["embed_tokens.weight"].to(BF16)
        self.norm = sd["norm.weight"].float()
        self.inv_freq = model.rotary_emb.inv_freq.float().to(self.device)
        self.blocks = []
        for i in range(c.num_hidden_layers):
            p = f"layers.{i}."
            w = {"in": sd[p + "input_layernorm.weight"].float(),
                 "post": sd[p + "post_attention_layernorm.weight"].float(),
                 "q": sd[p + "self_attn.q_norm.weight"].float(), "k": sd[p + "self_attn.k_norm.weight"].float(),
                 "o": sd[p + "self_attn.o_proj.weight"].to(BF16).contiguous(),
                 "down": sd[p + "mlp.down_proj.weight"].to(BF16).contiguous()}
            qkv = torch.cat([sd[p + f"self_attn.{x}_proj.weight"] for x in "qkv"]).to(BF16)
            up = torch.cat([sd[p + "mlp.gate_proj.weight"], sd[p + "mlp.up_proj.weight"]]).to(BF16)
            w["qkv"], w["up"] = (MXO.quant(qkv), MXO.quant(up)) if fp8 else (qkv, up)
            self.blocks.append(w)

    def _norm(self, delta, s, w):
        f = N.add_rms_fwd_mx if self.fp8 else N.add_rms_fwd
        h, s, _ = f(delta, s, w, self.eps)
        return h, s

    def _heads(self, x, w, cos, sin):
        """Per-head RMSNorm and RoPE (rotated halves) of [T, n * D]."""
        T, D = x.shape[0], self.head_dim
        x = x.view(T, -1, D).float()
        x = (x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + self.eps)).to(BF16).float() * w
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(BF16).view(T, -1)

    @torch.no_grad()
    def extend(self, cache, ids, new):
        """Appends packed token ids [sum(new)] (new[b] tokens to sequence b) and returns their final hidden states
        [sum(new), hidden] bf16."""
        dev, D = self.device, self.head_dim
        if len(new) != len(cache.lens) or ids.shape != (sum(new),):
            raise ValueError(f"{len(cache.lens)} counts that add up to the {tuple(ids.shape)} ids expected, got {new}")
        if min(new, default=0) < 0:
            raise ValueError(f"counts of new tokens expected, got {new}")
        total = [n + t for n, t in zip(new, cache.lens)]
        if max(total, default=0) > cache.max_tokens:
            raise ValueError(f"a sequence of {max(total)} tokens in a cache of {cache.max_tokens} each")
        if not sum(new):
            return self.embed.new_empty(0, self.embed.shape[1])
        counts = torch.tensor([cache.lens, new, total], dtype=torch.int32).to(dev)
        pos, tot = counts[0], counts[2]
        cu = torch.zeros(len(new) + 1, dtype=torch.int32, device=dev)
        cu[1:] = counts[1].cumsum(0)
        at = torch.cat([torch.arange(t, t + n) for n, t in zip(new, cache.lens)]).to(dev)
        ang = torch.outer(at.float(), self.inv_freq)
        cos, sin = ang.cos()[:, None], ang.sin()[:, None]
        Cq, Ck = self.heads * D, self.kv_heads * D
        lin = MXO.linear if self.fp8 else G.linear
        glu = MXO.swiglu_linear if self.fp8 else G.swiglu_linear
        delta = self.embed[ids.to(dev)]
        s = torch.zeros_like(delta)
        for w, kv in zip(self.blocks, cache.layers):
            h, s = self._norm(delta, s, w["in"])
            qkv = lin(h, w["qkv"])
            q = self._heads(qkv[:, :Cq], w["q"], cos, sin)
            k = self._heads(qkv[:, Cq:Cq + Ck], w["k"], cos, sin)
            P.cache_write(kv, k, qkv[:, Cq + Ck:], cache.table, pos, cu)
            o, _ = P.paged_attn(q, kv, cache.table, tot, cu, max(new), max(total))
            delta = G.linear(o, w["o"])
            h, s = self._norm(delta, s, w["post"])
            delta = G.linear(glu(h, w["up"])[0], w["down"])
        cache.lens = total
        return N.add_rms_fwd(delta, s, self.norm, self.eps)[0]

    @torch.no_grad()
    def encode(self, ids, mask, kind="bf16", chunk=None):
        """Final hidden states [B, L, hidden] bf16 of a left-aligned batch (zeros where mask is False), the keys and
        values in a cache of `kind`, `chunk` tokens of every sequence at a time (None: all at once)."""
        ids, mask = ids.cpu(), mask.cpu().bool()
        if (mask[:, 1:] & ~mask[:, :-1]).any():  # the tokens' positions would not be the columns
            raise ValueError("TextLM: a left-aligned mask expected (each row: its tokens, then padding)")
        if chunk is not None and chunk < 1:
            raise ValueError(f"chunk must be None or positive, got {chunk}")
        lens = mask.sum(1).tolist()
        cache = TextCache(self, len(lens), max(lens + [1]), kind)
        out = torch.zeros(*ids.shape, self.embed.shape[1], dtype=BF16, device=self.device)
        step = max(lens + [1]) if chunk is None else chunk
        for t in range(0, max(lens + [0]), step):
            part = torch.zeros_like(mask)
            part[:, t:t + step] = mask[:, t:t + step]
            out[part.to(self.device)] = self.extend(cache, ids[part], part.sum(1).tolist())
        return out
