"""Wrapped models on `tp.paged.PagedCache` between their steps: copies, held steps without positions, steps that fail, sequences that end under a captured forward, and generated tokens.

Tolerances of logits are those of test_gpu_paged_model.py."""
import copy

import pytest
import torch

import tensor_parallel_amd as tp
from test_gpu_paged_model import DEV, llama

pytestmark = pytest.mark.gpu


def fused(ranks, assume=True):
    model = tp.tensor_parallel(llama(torch.bfloat16), [DEV] * ranks)
    tp.attention.fuse_rotary_(model, assume_no_padding=assume)
    return model


def tokens(*shape, seed):
    return torch.randint(2, 300, shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


def step(model, cache, ids, counts=None, **more):
    positions = {"position_ids": cache.prepare(counts, **more).to(DEV)} if counts is not None else {}
    return model(input_ids=ids, past_key_values=cache, use_cache=True, **positions).logits


@pytest.mark.parametrize("ranks", [1, 2])
def test_a_prefix_is_continued_in_two_ways(ranks):
    """A copy goes on from the prompt as a cache that was given the prompt itself does, and neither disturbs the other."""
    model, prompt, ways = fused(ranks), tokens(2, 50, seed=1), [tokens(3, 2, 1, seed=2), tokens(3, 2, 1, seed=3)]
    caches = [tp.paged.PagedCache(sequences=2, pages=16, page=16) for _ in "ab"]
    with torch.no_grad():
        for cache in caches:
            step(model, cache, prompt, [50, 31])
        shared = copy.deepcopy(caches[0])
        for i in range(3):
            for cache, way in ((caches[0], ways[0]), (shared, ways[1]), (caches[1], ways[1])):
                out = step(model, cache, way[i], [1, 1])
                if cache is shared:
                    kept = out.clone()
            assert torch.equal(kept, out)
    assert [c.lengths() for c in (*caches, shared)] == [[53, 34]] * 3


def test_held_forwards_without_positions_are_the_one_with_them():
    model, prompt, token = fused(2), tokens(2, 50, seed=4), tokens(2, 1, seed=5)
    cache = tp.paged.PagedCache(sequences=2, pages=16, page=16)
    with torch.no_grad():
        step(model, cache, prompt)
        want = step(model, cache, token, [1, 1], hold=True).clone()
        for _ in range(3):
            assert torch.equal(step(model, cache, token), want)
    assert cache.lengths() == [51, 51]


def test_a_forward_that_failed_is_made_again():
    model, prompt, token = fused(1), tokens(2, 50, seed=6), tokens(2, 1, seed=7)
    caches = [tp.paged.PagedCache(sequences=2, pages=16, page=16) for _ in "ab"]
    mlp = [m for m in model.modules() if type(m).__name__ == "LlamaMLP"][0]

    def fails(*_):
        raise MemoryError("on the way")

    with torch.no_grad():
        for cache in caches:
            step(model, cache, prompt, [50, 31])
        want = step(model, caches[1], token, [1, 1])
        for prepared in (True, False):
            hook = mlp.register_forward_pre_hook(fails)
            with pytest.raises(MemoryError):
                step(model, caches[0], token, [1, 1])
            hook.remove()
            caches[0].abandon()
            assert caches[0].lengths() == [50, 31]
        assert torch.equal(step(model, caches[0], token, [1, 1]), want)


def test_replays_after_a_release_leave_the_pages_alone():
    model, prompt, token = fused(2), tokens(2, 50, seed=8), tokens(2, 1, seed=9)
    cache = tp.paged.PagedCache(sequences=2, pages=16, page=16)
    with torch.no_grad():
        step(model, cache, prompt, [50, 31])
        with pytest.raises(ValueError, match="hold"):
            tp.graphs.capture(model, input_ids=token, position_ids=torch.tensor([[50], [31]], device=DEV), past_key_values=cache, use_cache=True)
        positions = cache.prepare([1, 1], hold=True).to(DEV)
        with pytest.raises(ValueError, match="position_ids"):
            tp.graphs.capture(model, input_ids=token, past_key_values=cache, use_cache=True)
        graph = tp.graphs.capture(model, input_ids=token, position_ids=positions, past_key_values=cache, use_cache=True)
        with pytest.raises(ValueError, match="rows"):
            cache.prepare([2, 1], hold=True)
        graph(input_ids=token, position_ids=positions, past_key_values=cache, use_cache=True)
        cache.release(0)
        pools = [p for c in tp.kv_cache.rank_caches(cache, 2) for layer in c._pools.values() for p in layer]
        before = [p.clone() for p in pools]
        for _ in range(3):
            graph(input_ids=token + 1, position_ids=positions, past_key_values=cache, use_cache=True)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(pools, before))
        # and a step that is prepared then is the eager one
        eager = copy.deepcopy(cache)
        want = step(model, eager, token, [1, 1])
        positions = cache.prepare([1, 1], hold=True).to(DEV)
        for _ in range(2):
            got = graph(input_ids=token, position_ids=positions, past_key_values=cache, use_cache=True).logits
            tol = 32 * torch.finfo(torch.bfloat16).eps / 2 * float(want.float().std())
            assert (got.float() - want.float()).abs().max() <= tol
            torch.cuda.synchronize()
    assert cache.lengths() == eager.lengths() == [1, 33]


def test_generated_tokens_are_the_likeliest():
    """Each token that `generate` chose on pages is, on a growing cache that is given all of them at once, within the two sides' tolerances of the likeliest one there."""
    from transformers import DynamicCache

    model, ids, new = fused(2), tokens(2, 50, seed=3), 12
    with torch.no_grad():
        out = model.generate(ids, attention_mask=torch.ones_like(ids), past_key_values=tp.paged.PagedCache(sequences=2, pages=16, page=16), max_new_tokens=new, do_sample=False)
        logits = model(input_ids=out[:, :-1], past_key_values=DynamicCache(), use_cache=True).logits[:, 49:].float()
    assert out.shape == (2, 62) and torch.equal(out[:, :50], ids)
    chosen = logits.gather(2, out[:, 50:, None])[..., 0]
    tol = 32 * torch.finfo(torch.bfloat16).eps / 2 * float(logits.std())
    assert (logits.max(-1).values - chosen).max() <= 2 * tol
    assert len(out[:, 50:].unique()) > 1
