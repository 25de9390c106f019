"""The graphed decode loop before the first full block: its steps depend on the context's
length on the host (dense attention), so they run eagerly; tokens and caches equal the eager
loop's from a prompt that is shorter than a block until past the first compression."""
import pytest
import torch

from conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]


@pytest.mark.parametrize("T", [8, 490, 511])
def test_graphed_equals_eager_from_a_short_prompt(T):
    from unsloth_spectral.llama_loop import LlamaShape, SpectralLlama
    shape = LlamaShape(layers=2, hidden=512, heads=8, kv_heads=2, head_dim=128, ffn=1024, vocab=1000)
    model = SpectralLlama(shape, device="cuda", dtype=torch.float16, std=0.05, seed=8)
    model.patch(block_size=512, k_rank_keys=16, k_rank_values=16)
    prompt = torch.randint(0, 1000, (2, T), generator=torch.Generator(device="cuda").manual_seed(T), device="cuda")
    new = 40 if T > 400 else 12
    runs = []
    for graphs in (False, True):
        torch.manual_seed(12)
        runs.append((model.generate(prompt, new, cuda_graphs=graphs), model._caches[1].hot_K.clone()))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])


def test_graphed_equals_eager_with_dense_attention():
    """Layers patched to keep dense attention past the first block."""
    from unsloth_spectral.llama_loop import LlamaShape, SpectralLlama
    shape = LlamaShape(layers=2, hidden=512, heads=8, kv_heads=2, head_dim=128, ffn=1024, vocab=1000)
    model = SpectralLlama(shape, device="cuda", dtype=torch.float16, std=0.05, seed=8)
    model.patch(block_size=512, k_rank_keys=16, k_rank_values=16, use_spectral_attention=False)
    prompt = torch.randint(0, 1000, (2, 530), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    runs = []
    for graphs in (False, True):
        torch.manual_seed(12)
        runs.append((model.generate(prompt, 12, cuda_graphs=graphs), model._caches[1].hot_K.clone()))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
