"""The transformers hook with ``rotary_kernel``: rotated prompts and steps of a randomly initialised Llama against the
same hook with the model's own rotation, over the same tokens.

Logits of the two differ by roundings of keys and queries (the model's rotation rounds its products to the model's
type, the kernel the exact sum once) and, through them, by a code of the cache here and there; a wrong position, pairing
or head order would leave no agreement.  The measure is the one that the hook's other tests use: the cosine of a
position's logits above 0.995."""

import pytest
import torch

transformers = pytest.importorskip("transformers")

from turbopolar_amd import llama as tl  # noqa: E402
from turbopolar_amd.fast_attention import TurboPolarFastCache  # noqa: E402

pytestmark = pytest.mark.gpu


def model_of(device, dtype):
    from transformers import LlamaConfig, LlamaForCausalLM

    cfg = LlamaConfig(vocab_size=512, hidden_size=1024, intermediate_size=1024, num_hidden_layers=2,
                      num_attention_heads=8, num_key_value_heads=2, head_dim=128, max_position_embeddings=4096,
                      attn_implementation="eager")
    torch.manual_seed(0)
    return LlamaForCausalLM(cfg).to(device=device, dtype=dtype).eval()


def steps(model, tokens, prompt, **patch):
    """Logits after a prompt, a chunk of five tokens and single steps, and the calls of ``decode_rotated``."""
    cache, calls, out = tl.make_turbo_cache(model), [0], []
    real = TurboPolarFastCache.decode_rotated

    def counted(self, *a, **k):
        calls[0] += 1
        return real(self, *a, **k)

    TurboPolarFastCache.decode_rotated = counted
    tl.patch_llama_attention(model, **patch)
    try:
        with torch.no_grad():
            at = 0
            while at < tokens.shape[1]:
                n = prompt if at == 0 else 5 if at == prompt else 1
                out.append(model(tokens[:, at:at + n], past_key_values=cache, use_cache=True).logits[:, -1])
                at += n
    finally:
        tl.unpatch_llama_attention(model)
        TurboPolarFastCache.decode_rotated = real
    assert cache.fast(0).offset == cache.fast(1).offset == tokens.shape[1]
    return torch.stack(out).double(), calls[0]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("prompt_kernel", [False, True])
def test_the_hook(device, dtype, prompt_kernel):
    model = model_of(device, getattr(torch, dtype))
    tokens = torch.randint(0, 512, (1, 150), generator=torch.Generator().manual_seed(1)).to(device)
    want, none = steps(model, tokens, 110, prompt_kernel=prompt_kernel)
    got, calls = steps(model, tokens, 110, prompt_kernel=prompt_kernel, rotary_kernel=True)
    assert none == 0 and calls == 2 * 35  # each layer's single tokens
    near = torch.nn.functional.cosine_similarity(got, want, dim=-1).min()
    print(f"[rotary] {dtype} prompt_kernel={prompt_kernel}: smallest cosine {float(near):.6f}", flush=True)
    assert torch.isfinite(got).all() and near > 0.995
    # Another position's logits are no match, so the measure means something.
    assert torch.nn.functional.cosine_similarity(got[1:], want[:-1], dim=-1).max() < 0.95


def test_gradients_take_the_models_rotation(device):
    """With gradients enabled nothing is turned by the kernel, which has no backward pass."""
    model = model_of(device, torch.float32)
    tokens = torch.randint(0, 512, (1, 12), generator=torch.Generator().manual_seed(2)).to(device)
    tl.patch_llama_attention(model, prompt_kernel=True, rotary_kernel=True)
    try:
        model(tokens).logits.sum().backward()
    finally:
        tl.unpatch_llama_attention(model)
    assert all(torch.isfinite(p.grad).all() for p in model.parameters())
