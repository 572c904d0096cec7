"""The serving operators at their edges: slots that were used before, calls that fail half way, sequences that end at a page's
border, pages that are shared, and numbers at the ends of their ranges.  CPU tensors take the PyTorch definitions; the
gpu-marked tests take the HIP kernels."""
import pytest
import torch

import paddle2_amd as paddle
from paddle2_amd import serving
from paddle2_amd.serving import LlamaGenerator

DEVS = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _llama(dev, **kw):
    from paddle2_amd.models import LlamaConfig, LlamaForCausalLM

    paddle.seed(3)
    kw.setdefault("dtype", "bfloat16" if dev == "cuda" else "float32")
    m = LlamaForCausalLM(LlamaConfig.tiny(num_attention_heads=4, num_key_value_heads=2, **kw))
    if dev == "cuda":
        paddle.set_device("gpu:0")
        m.to(device="gpu:0")
    m.eval()
    return m


def _near(dev):
    return dict(atol=3e-2, rtol=3e-2) if dev == "cuda" else dict(atol=1e-4, rtol=1e-4)


# ============================================================================ prompts over slots that were used before
@pytest.mark.parametrize("dev", DEVS)
def test_chunked_prompts_start_at_zero_in_used_slots(dev):
    """A prompt in pieces replaces what its slot holds, as prefill does."""
    m = _llama(dev)
    prompts = [[1, 5, 9, 3, 11, 4, 8, 2, 6], [7, 2, 8]]
    gen = LlamaGenerator(m, max_batch=2, max_seq_len=64, block_size=8, use_graph=False)
    fresh = gen.prefill_chunks([0, 1], prompts, 4).clone()
    gen.cache.free(0), gen.cache.free(1)
    for s in (0, 1):
        gen.prefill(s, torch.arange(30, 47))
    again = gen.prefill_chunks([0, 1], prompts, 4)
    assert torch.equal(again, fresh) and gen.cache.seq_lens.tolist() == [9, 3]


def test_chunked_generation_after_an_earlier_prompt_and_a_failed_call():
    m = _llama("cpu")
    prompts = [[1, 5, 9, 3, 11, 4, 8, 2, 6], [7, 2, 8]]
    gen = LlamaGenerator(m, max_batch=2, max_seq_len=64, block_size=8, use_graph=False)
    plain = gen.generate(prompts, 6)
    assert gen.generate(prompts, 6, chunk_size=4) == plain
    gen.prefill(0, torch.arange(30, 47))
    assert gen.generate(prompts, 6, chunk_size=4) == plain
    with pytest.raises(IndexError):
        gen.generate([[3] * 20], 60, chunk_size=4)
    assert gen.generate(prompts, 6, chunk_size=4) == plain


# ============================================================================ calls that fail half way
def test_generate_that_fails_leaves_its_slots_free():
    """Out of room after the pages were forked, in the prompt, or at the draw: the slots are free and the next call works."""
    m = _llama("cpu")
    gen = LlamaGenerator(m, max_batch=2, max_seq_len=64, block_size=8, use_graph=False)
    plain = gen.generate([[1, 2, 3]], 6)
    for err, f in ((IndexError, lambda: gen.generate([list(range(1, 18))], 60, num_return_sequences=2)),
                   (IndexError, lambda: gen.generate([[4] * 70, [1]], 2)),
                   (ValueError, lambda: gen.generate([[1, 2]], 3, temperature=-1.0, sampler="fused"))):
        with pytest.raises(err):
            f()
        assert gen.cache.num_free_blocks == len(gen.cache._holders) and gen.cache.seq_lens.tolist() == [0, 0]
        assert gen.generate([[1, 2, 3]], 6) == plain


def test_generate_that_is_refused_changes_nothing():
    """Bad arguments, and continuations whose slots hold something, are refused before anything is computed."""
    gen = LlamaGenerator(_llama("cpu"), max_batch=3, max_seq_len=64, block_size=8, use_graph=False)
    gen.prefill(1, torch.arange(5, 16))
    pools = [t.clone() for t in gen.cache.k + gen.cache.v]
    calls = []
    gen._layer_qkv = lambda *a: calls.append(a)
    for f in (lambda: gen.generate([[1, 2]], 2, num_return_sequences=2), lambda: gen.generate([[1, 2]], 2, chunk_size=0),
              lambda: gen.generate([[1, 2], []], 2, chunk_size=4), lambda: gen.generate([[1, 2]], 2, top_k=[1, 2])):
        with pytest.raises(ValueError):
            f()
    assert not calls and gen.cache.seq_lens.tolist() == [0, 11, 0] and len(gen.cache._owned[1]) == 2
    assert all(torch.equal(a, b) for a, b in zip(pools, gen.cache.k + gen.cache.v))
