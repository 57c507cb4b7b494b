"""Scoring a continuation through the plugin backends: run_score against run_decode's logits, and
the packed backend's chunks (several new tokens over the packed far segment) against one token
at a time."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(device, hd=64, dtype=torch.float32):
    from transformers import GPT2Config, GPT2LMHeadModel
    cfg = GPT2Config(n_layer=2, n_head=4, n_embd=4 * hd, vocab_size=300, n_positions=512)
    torch.manual_seed(3)
    return (GPT2LMHeadModel(cfg).eval().to(device).to(dtype),
            dict(n_layers=2, n_kv_heads=4, head_dim=hd))


def _ids(device, n, batch=1, seed=5):
    return torch.randint(0, 300, (batch, n), generator=torch.Generator().manual_seed(seed)).to(device)


@pytest.mark.parametrize("name", ["dense", "quant_int4", "quant_packed"])
@pytest.mark.parametrize("batch", [1, 2])
def test_scores_are_those_of_run_decode(name, batch, cuda_device):
    from knlp_b200 import backends as B
    model, mc = _model(cuda_device)
    prefix, cont = _ids(cuda_device, 120, batch), _ids(cuda_device, 9, batch, 6)
    b = B.get_backend(name)
    b.configure(120, mc, W_min=32, W_sink=4)
    b.calibrated, b.layer_bits = True, [4, 8]
    logits, _ = b.run_decode(model, prefix, cont, str(cuda_device), 512)
    for chunk in ((1, 4, 256) if name == "quant_packed" else (None,)):
        kw = {} if chunk is None else dict(chunk=chunk)
        s, stats = b.run_score(model, prefix, cont, str(cuda_device), 512, top_k=3, **kw)
        want = torch.log_softmax(logits[:, :-1].double(), -1)
        lp = want.gather(-1, cont[..., None])[..., 0]
        assert s.logprob.shape == (batch, 9) and s.top_ids.shape == (batch, 9, 3)
        # chunk 1 and the other backends: the same logits; chunks: attention within the decode
        # kernels' bar (2e-3 + 1e-3 |o|), which the two layers and the head carry to the logits
        tol = 1e-5 if chunk in (None, 1) else 1e-2
        assert (s.logprob.double() - lp).abs().max() < tol
        ent = -(want.exp() * want).sum(-1)
        assert (s.entropy.double() - ent).abs().max() < tol
        assert len(stats) == (9 if chunk in (None, 1) else -(-9 // chunk))
        assert stats[-1].kv_kept == 129
        if name == "quant_packed":
            assert stats[0].n_compressed == 84 and stats[-1].n_full == 36 + 9
            assert model.config._attn_implementation != "knlp_b200_packed"
    s, _ = b.run_score(model, prefix, cont, str(cuda_device), 512)
    assert s.rank.shape == (batch, 9) and s.top_ids.shape == (batch, 9, 0)


def test_short_inputs_and_refusals(cuda_device):
    from knlp_b200 import backends as B
    model, mc = _model(cuda_device)
    b = B.get_backend("quant_packed")
    b.configure(30, mc, W_min=32, W_sink=4)  # nothing far: the dense part alone
    prefix, cont = _ids(cuda_device, 30), _ids(cuda_device, 5, seed=6)
    s, stats = b.run_score(model, prefix, cont, str(cuda_device), 512, chunk=3)
    d = B.get_backend("dense")
    d.configure(30, mc)
    t, _ = d.run_score(model, prefix, cont, str(cuda_device), 512)
    assert (s.logprob - t.logprob).abs().max() < 1e-3 and stats[0].n_compressed == 0
    s, stats = b.run_score(model, prefix, cont[:, :0], str(cuda_device), 512)
    assert s.logprob.shape == (1, 0) and stats == []
    with pytest.raises(ValueError):
        b.run_score(model, prefix, cont, str(cuda_device), 512, chunk=0)
    with pytest.raises(ValueError):  # and the model has its own attention again
        b.run_score(model, prefix, cont, str(cuda_device), 512, top_k=1000)
    assert model.config._attn_implementation != "knlp_b200_packed"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [1, 7, 40])
def test_packed_attention_of_several_tokens(T, dtype, cuda_device):
    """The attention function alone, against softmax in 64 bits over the far and the full tokens.
    Bound: 16-bit rounding of the result, and of P, V and (through the scores) K, each within 2^-11
    of its value: |o| 2^-8 (bf16) + (2 e + 2^-9) max |v| with e = scale max sum |q k| 2^-10."""
    from types import SimpleNamespace
    from knlp_b200 import backends as B
    from knlp_b200.cache import PackedKVCache
    dev, b, h, hkv, d, far, near = cuda_device, 2, 4, 2, 64, 150, 20
    g = torch.Generator(device=dev).manual_seed(T)
    rand = lambda *s: torch.randn(s, generator=g, device=dev).to(dtype)
    c = PackedKVCache(hkv, d, "int8", "int8")
    pages = -(-far // 16)
    c.ensure(b * pages, 16, dev)
    table = torch.arange(b * pages, dtype=torch.int32, device=dev).view(b, pages)
    pos = torch.arange(far, device=dev)
    slots = (table[:, pos // 16].long() * 16 + pos % 16).reshape(-1)
    c.write(rand(b * far, hkv, d), rand(b * far, hkv, d), slots)
    values = lambda codes, sc: (codes.double() * sc.double().repeat_interleave(32, -1)).view(
        -1, hkv, d)[slots].view(b, far, hkv, d).transpose(1, 2)
    q, k, v = rand(b, h, T, d), rand(b, hkv, near + T, d), rand(b, hkv, near + T, d)
    state = SimpleNamespace(_far=[(c, table, torch.full((b,), far, dtype=torch.int32, device=dev))],
                            _n_far=far)
    B._ACTIVE_PACKED = state
    try:
        out, _ = B._packed_attention(SimpleNamespace(layer_idx=0), q, k, v)
    finally:
        B._ACTIVE_PACKED = None
    ka = torch.cat([values(c.key_cache, c.k_scales), k.double()], 2).repeat_interleave(2, 1)
    va = torch.cat([values(c.value_cache, c.v_scales), v.double()], 2).repeat_interleave(2, 1)
    w = q.double() @ ka.transpose(2, 3) * d ** -0.5
    e = (q.double().abs() @ ka.abs().transpose(2, 3)).amax() * d ** -0.5 * 2.0 ** -10
    off = torch.arange(far + near + T, device=dev)[None] > far + near + torch.arange(T, device=dev)[:, None]
    want = (torch.softmax(w.masked_fill(off, float("-inf")), -1) @ va).transpose(1, 2)
    bound = want.abs() * torch.finfo(dtype).eps / 2 + (2 * e + 2.0 ** -9) * va.abs().amax()
    assert out.shape == (b, T, h, d) and ((out.double() - want).abs() <= bound).all()
