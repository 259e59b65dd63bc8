"""What models/text_lm.py refuses, and how the conditioner keeps it in step with its module."""
import pytest
import torch


def _qwen3(**kw):
    transformers = pytest.importorskip("transformers")
    torch.manual_seed(0)
    c = dict(vocab_size=97, hidden_size=128, intermediate_size=256, num_hidden_layers=2, num_attention_heads=2,
             num_key_value_heads=1, head_dim=64, max_position_embeddings=256)
    c.update(kw)
    m = transformers.Qwen3Model(transformers.Qwen3Config(**c)).eval()
    for p in m.parameters():
        if p.dim() == 2:
            p.data.copy_(p.data.bfloat16().float() * 3)
    return m


@pytest.mark.parametrize("kw,what", [
    ({"attention_bias": True}, "bias"),
    ({"use_sliding_window": True, "sliding_window": 16, "max_window_layers": 0}, "sliding window"),
    ({"use_sliding_window": True, "sliding_window": 16, "max_window_layers": 1}, "sliding window"),
    ({"hidden_act": "gelu"}, "hidden_act"),
    ({"rope_scaling": {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64}}, "rotary"),
    ({"rope_scaling": {"rope_type": "dynamic", "factor": 2.0}}, "rotary")])
def test_a_model_that_the_blocks_do_not_compute_is_refused(kw, what):
    from nano_gpic_b200.models.conditioner import Qwen3TextEncoder
    from nano_gpic_b200.models.text_lm import TextLM
    m = _qwen3(**kw)
    with pytest.raises(ValueError, match=what):
        TextLM(m)
    with pytest.raises(ValueError, match=what):
        Qwen3TextEncoder(model=m, tokenizer=lambda *a, **k: None, native="bf16")


@pytest.mark.parametrize("kw", [{}, {"use_sliding_window": True, "sliding_window": 16, "max_window_layers": 2},
                                {"rope_scaling": {"rope_type": "linear", "factor": 2.0}}])
def test_what_they_do_compute_is_accepted(kw):
    """Against transformers in fp32; tolerance as in test_text_lm.py for bf16."""
    from nano_gpic_b200.models.text_lm import TextLM
    m = _qwen3(**kw)
    ids = torch.randint(0, 97, (2, 40), generator=torch.Generator().manual_seed(1))
    mask = torch.ones_like(ids, dtype=torch.bool)
    with torch.no_grad():
        ref = m(input_ids=ids, attention_mask=mask.long())[0]
    d = TextLM(m).encode(ids, mask).float() - ref
    assert d.square().mean().sqrt() <= 0.02 * ref.square().mean().sqrt()


def _captions():
    ids = torch.randint(0, 97, (3, 24), generator=torch.Generator().manual_seed(2))
    return ids, torch.arange(24)[None] < torch.tensor([24, 1, 9])[:, None]


def _encoder(m, **kw):
    from nano_gpic_b200.models.conditioner import Qwen3TextEncoder
    return Qwen3TextEncoder(model=m, tokenizer=lambda *a, **k: None, native="bf16", **kw)


def test_native_encoder_follows_the_weights():
    ids, mask = _captions()
    enc, other = _encoder(_qwen3()), _qwen3()
    old, _ = enc.encode(ids, mask)
    for p in other.parameters():
        p.data.mul_(1.25)
    enc.model.load_state_dict(other.state_dict())
    got, _ = enc.encode(ids, mask)
    want, _ = _encoder(other).encode(ids, mask)
    assert torch.equal(got, want) and not torch.equal(got, old)
    assert enc.lm is enc.lm  # laid out once


@pytest.mark.gpu
def test_native_encoder_follows_the_module_to_another_device():
    ids, mask = _captions()
    enc = _encoder(_qwen3())
    enc.encode(ids, mask)
    got, _ = enc.to("cuda").encode(ids, mask)
    want, _ = _encoder(_qwen3(), device="cuda").encode(ids, mask)
    assert got.is_cuda and torch.equal(got, want)


def test_a_mask_that_is_not_left_aligned_is_refused():
    from nano_gpic_b200.models.text_lm import TextLM
    lm = TextLM(_qwen3())
    ids, mask = _captions()
    for bad in (mask.flip(1), torch.cat([mask[:, :3], mask[:, :3]], 1) & torch.tensor([1, 0, 1, 1, 1, 1]).bool()):
        with pytest.raises(ValueError, match="left-aligned"):
            lm.encode(ids[:, :bad.shape[1]], bad)
    assert lm.encode(ids[:, :0], mask[:, :0]).shape == (3, 0, 128)


def test_negative_counts_and_chunks_are_refused():
    from nano_gpic_b200.models.text_lm import TextCache, TextLM
    lm = TextLM(_qwen3())
    ids, mask = _captions()
    for chunk in (0, -5):
        with pytest.raises(ValueError, match="chunk"):
            lm.encode(ids, mask, chunk=chunk)
    cache = TextCache(lm, 2, 8)
    with pytest.raises(ValueError, match="counts"):
        lm.extend(cache, ids[0, :2], [3, -1])
    assert cache.lens == [0, 0]


def _at_head_dim_128(dev, kind, chunk, lim):
    from nano_gpic_b200.models.text_lm import TextLM
    m = _qwen3(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=128)
    ids = torch.randint(0, 97, (3, 150), generator=torch.Generator().manual_seed(3))
    mask = torch.arange(150)[None] < torch.tensor([150, 1, 77])[:, None]
    with torch.no_grad():
        ref = m(input_ids=ids, attention_mask=mask.long())[0]
    out = TextLM(m.to(dev)).encode(ids.to(dev), mask.to(dev), kind=kind, chunk=chunk).float().cpu()
    d, r = (out - ref)[mask], ref[mask]
    assert (out[~mask] == 0).all() and d.square().mean().sqrt() <= lim * r.square().mean().sqrt()


# heads of 128, the encoder's own; tolerances as in test_text_lm.py
CASES_128 = [("bf16", None, 0.02), ("bf16", 50, 0.02), ("e4m3", None, 0.1)]


@pytest.mark.parametrize("kind,chunk,lim", CASES_128)
def test_head_dim_128_cpu(kind, chunk, lim):
    _at_head_dim_128("cpu", kind, chunk, lim)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,chunk,lim", CASES_128 + [("bf16", 1, 0.02), ("e4m3", 8, 0.1)])
def test_head_dim_128_gpu(kind, chunk, lim):
    from nano_gpic_b200.ops import status
    _at_head_dim_128("cuda", kind, chunk, lim)
    status.check()


def test_a_config_without_layer_types():
    from nano_gpic_b200.models.text_lm import check_model
    m = _qwen3()
    m.config.layer_types = None
    check_model(m)
    m.config.use_sliding_window = True
    with pytest.raises(ValueError, match="sliding window"):
        check_model(m)
