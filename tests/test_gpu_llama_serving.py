"""The transformers Llama hook's prompt kernel and its cache protocol on the GPU: prompts and chunks
through tp_prompt_attention against the model's own attention over the same compressed history, and
crop / select / repeat against caches that never held what was removed."""

import pytest
import torch

transformers = pytest.importorskip("transformers")

from turbopolar_amd import llama as tl  # noqa: E402
from turbopolar_amd.fast_attention import TurboPolarFastCache  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    from transformers import LlamaConfig, LlamaForCausalLM

    if not torch.cuda.is_available():
        pytest.skip("no HIP device in this environment")
    cfg = LlamaConfig(vocab_size=512, hidden_size=1024, intermediate_size=1024, num_hidden_layers=2,
                      num_attention_heads=8, num_key_value_heads=2, head_dim=128, max_position_embeddings=4096,
                      attn_implementation="eager")
    torch.manual_seed(0)
    return LlamaForCausalLM(cfg).to(device="cuda:0", dtype=torch.bfloat16).eval()


def _logits(model, ids, cache):
    with torch.no_grad():
        return model(ids, past_key_values=cache, use_cache=True).logits


def _tokens(B, T, seed):
    return torch.randint(0, 512, (B, T), generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("B", [1, 2])
def test_prompt_kernel_matches_the_models_attention(model, B, monkeypatch):
    """Chunks of 100, 1 (batch 1: the decode kernel) and 90 tokens.  Both runs read the same kind of
    compressed history; the model's own attention rounds scores and weights to bfloat16, so logits
    agree as its steps of 2^-8 let them."""
    ids = _tokens(B, 191, 1)
    calls = []
    orig = TurboPolarFastCache.prompt_attention
    monkeypatch.setattr(TurboPolarFastCache, "prompt_attention", lambda self, *a, **k: (calls.append(1), orig(self, *a, **k))[1])
    chunks = [ids[:, :100], ids[:, 100:101], ids[:, 101:]] if B == 1 else [ids[:, :100], ids[:, 100:]]
    got, want = [], []
    ours, theirs = tl.make_turbo_cache(model), tl.make_turbo_cache(model)
    try:
        tl.patch_llama_attention(model, prompt_kernel=True)
        got = [_logits(model, c, ours) for c in chunks]
        assert len(calls) == 2 * 2 and ours.get_seq_length() == 191
        tl.patch_llama_attention(model)  # the default: prompts are the model's
        want = [_logits(model, c, theirs) for c in chunks]
        assert len(calls) == 4
    finally:
        tl.unpatch_llama_attention(model)
    for a, b in zip(got, want):
        a, b = a.double().flatten(), b.double().flatten()
        cos = float((a @ b) / (a.norm() * b.norm()))
        print(f"[llama] prompt kernel cosine {cos:.6f}", flush=True)
        assert cos >= 0.999


def test_padded_batch_keeps_the_models_attention(model, monkeypatch):
    """A mask that is not the full causal one is not the kernel's."""
    monkeypatch.setattr(TurboPolarFastCache, "prompt_attention", lambda *a, **k: pytest.fail("called"))
    ids, mask = _tokens(2, 12, 2), torch.ones((2, 12), dtype=torch.long, device="cuda:0")
    mask[0, :5] = 0
    try:
        tl.patch_llama_attention(model, prompt_kernel=True)
        with torch.no_grad():
            out = model(ids, attention_mask=mask, past_key_values=tl.make_turbo_cache(model), use_cache=True).logits
        assert torch.isfinite(out[:, -1]).all()
    finally:
        tl.unpatch_llama_attention(model)


def test_crop_and_select(model):
    """A cache cropped inside its dense tail, or re-ordered, goes on like one that never held the rest."""
    ids = _tokens(2, 90, 3)
    one, two = tl.make_turbo_cache(model), tl.make_turbo_cache(model)
    _logits(model, ids[:, :80], one)
    _logits(model, ids[:, 80:], one)
    one.crop(-10)
    _logits(model, ids[:, :80], two)
    assert one.get_seq_length() == two.get_seq_length() == 80
    more = _tokens(2, 7, 4)
    assert torch.equal(_logits(model, more, one), _logits(model, more, two))
    one.crop(80)
    two.crop(-7)
    one.crop(200)  # longer than the cache: nothing
    assert one.get_seq_length() == two.get_seq_length() == 80
    for layer in range(2):
        assert torch.equal(one.fast(layer).runtime.partial_k, two.fast(layer).runtime.partial_k)
    one.reorder_cache(torch.tensor([1, 0], device="cuda:0"))
    swapped, straight = _logits(model, more[[1, 0]], one), _logits(model, more, two)
    assert torch.equal(swapped[[1, 0]], straight)
    one.batch_repeat_interleave(2)
    assert one.fast(0).runtime._batch_size == 4
    one.batch_select_indices(torch.tensor([True, False, False, True], device="cuda:0"))
    assert torch.equal(_logits(model, more[:, :3], one), _logits(model, more[:, :3], _rebuilt(model, ids, more)))
    empty = tl.make_turbo_cache(model)
    empty.crop(-3)
    empty.reorder_cache(torch.tensor([0], device="cuda:0"))
    assert empty.get_seq_length() == 0


def _rebuilt(model, ids, more):
    """The rows [1, 0] of the 80 tokens and the 7 after them, as the re-ordered cache holds them."""
    cache = tl.make_turbo_cache(model)
    _logits(model, ids[[1, 0], :80], cache)
    _logits(model, more[[1, 0]], cache)
    return cache


def test_assisted_generation(model):
    """Prompt-lookup generation drafts, verifies and crops on the compressed cache."""
    ids = torch.cat([_tokens(1, 20, 5)] * 3, 1)
    try:
        tl.patch_llama_attention(model)
        args = dict(max_new_tokens=12, do_sample=False, use_cache=True, pad_token_id=0)
        out = model.generate(ids, past_key_values=tl.make_turbo_cache(model), prompt_lookup_num_tokens=4, **args)
    finally:
        tl.unpatch_llama_attention(model)
    assert out.shape[0] == 1 and 61 <= out.shape[1] <= 72 and torch.equal(out[:, :60], ids)


@pytest.mark.parametrize("by", ["call", "config"])
def test_attention_weights_are_the_models(model, by, monkeypatch):
    """A step that asks for the attention's weights, by its call or by the configuration, gets them."""
    ids = _tokens(1, 20, 6)
    asked = dict(output_attentions=True) if by == "call" else {}
    if by == "config":
        monkeypatch.setattr(model.config, "output_attentions", True)
    try:
        tl.patch_llama_attention(model, prompt_kernel=True)
        cache = tl.make_turbo_cache(model)
        with torch.no_grad():
            out = model(ids[:, :13], past_key_values=cache, use_cache=True, **asked)
            more = model(ids[:, 13:], past_key_values=cache, use_cache=True, **asked)
    finally:
        tl.unpatch_llama_attention(model)
    for weights, T, held in ((out.attentions, 13, 13), (more.attentions, 7, 20)):
        assert [w.shape for w in weights] == [(1, 8, T, held)] * 2
        assert all(((w.float().sum(-1) - 1).abs() <= held * 2.0 ** -8).all() for w in weights)  # bf16 weights of at most 1


def test_other_keywords_are_the_models(model, monkeypatch):
    """Sequences packed by their lengths, and attention without the causal mask, are not the kernel's."""
    monkeypatch.setattr(TurboPolarFastCache, "prompt_attention", lambda *a, **k: pytest.fail("called"))
    ids = _tokens(1, 12, 7)
    try:
        tl.patch_llama_attention(model, prompt_kernel=True)
        starts = torch.tensor([0, 5, 12], dtype=torch.int32, device="cuda:0")
        for asked in (dict(is_causal=False), dict(cu_seq_lens_q=starts, cu_seq_lens_k=starts)):
            with torch.no_grad():
                model(ids, past_key_values=tl.make_turbo_cache(model), use_cache=True, **asked)
    finally:
        tl.unpatch_llama_attention(model)


def test_inference_mode(model):
    """A prompt, a chunk, a step and a crop in inference mode are those of no_grad."""
    ids = _tokens(1, 80, 8)
    try:
        tl.patch_llama_attention(model, prompt_kernel=True)
        got, want = [], []
        for mode, out in ((torch.inference_mode, got), (torch.no_grad, want)):
            cache = tl.make_turbo_cache(model)
            with mode():
                for a, b in ((0, 60), (60, 75), (75, 76)):
                    out.append(model(ids[:, a:b], past_key_values=cache, use_cache=True).logits.clone())
                cache.crop(-70)
                out.append(model(ids[:, 6:], past_key_values=cache, use_cache=True).logits.clone())
    finally:
        tl.unpatch_llama_attention(model)
    assert cache.get_seq_length() == 80 and all(torch.equal(a, b) for a, b in zip(got, want))
