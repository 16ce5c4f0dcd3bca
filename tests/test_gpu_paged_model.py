"""Wrapped models on `tp.paged.PagedCache`: sequences of different lengths in one batch against each of them alone on a growing cache.

The layers' arithmetic differs in roundings: the rotation is rounded once instead of three times, probabilities against other references, products of other numbers of rows in other orders. Each is a few
half steps (2^-8 in bf16, 2^-11 in fp16) of values whose spread the norms keep; 8 of them per layer and part of the residual stream, two layers, bound them by 2 * 2 * 8 half steps of the logits' spread."""
from copy import deepcopy

import pytest
import torch

import tensor_parallel_amd as tp

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def llama(dtype, head_dim=64):
    from transformers import LlamaConfig, LlamaForCausalLM

    name = tp.attention.register()
    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=300, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=head_dim,
                      max_position_embeddings=2048, attn_implementation="eager", bos_token_id=1, eos_token_id=None, pad_token_id=0)
    model = LlamaForCausalLM(cfg).to(dtype).eval()
    model.config._attn_implementation = name
    return model


def falcon():
    from transformers import FalconConfig, FalconForCausalLM

    torch.manual_seed(1)
    cfg = FalconConfig(vocab_size=300, hidden_size=256, num_hidden_layers=2, num_attention_heads=4, num_kv_heads=2, new_decoder_architecture=True, alibi=False, bias=False,
                       bos_token_id=1, eos_token_id=None, pad_token_id=0, attn_implementation="eager")
    return FalconForCausalLM(cfg).to(torch.bfloat16).eval()


def close(got, want, dtype):
    tol = 32 * torch.finfo(dtype).eps / 2 * float(want.float().std())
    assert (got.float() - want.float()).abs().max() <= tol


def padded(rows):
    width = max(len(r) for r in rows)
    return torch.tensor([r + [0] * (width - len(r)) for r in rows]).to(DEV)


PROMPTS = [40, 7, 100]


def alone(model, tokens, prompts):
    """Logits of each sequence's prompt and further tokens, one sequence at a time on a growing cache."""
    from transformers import DynamicCache

    outs = []
    for row, n in zip(tokens, prompts):
        cache = DynamicCache()
        out = [model(input_ids=torch.tensor([row[:n]]).to(DEV), past_key_values=cache, use_cache=True).logits[0]]
        for token in row[n:]:
            out.append(model(input_ids=torch.tensor([[token]]).to(DEV), past_key_values=cache, use_cache=True).logits[0])
        outs.append(torch.cat(out))
    return outs


@pytest.mark.parametrize("ranks", [1, 2])
@pytest.mark.parametrize("make,dtype,assume", [(lambda: llama(torch.bfloat16), torch.bfloat16, False), (lambda: llama(torch.float16, 128), torch.float16, False), (falcon, torch.bfloat16, True)])
def test_ragged_sequences_are_each_alone(ranks, make, dtype, assume):
    model = tp.tensor_parallel(make(), [DEV] * ranks)
    assert tp.attention.fuse_rotary_(model, assume_no_padding=assume) == 2 * ranks
    g = torch.Generator().manual_seed(2)
    steps = 5
    tokens = [torch.randint(2, 300, (n + steps,), generator=g).tolist() for n in PROMPTS]
    cache = tp.paged.PagedCache(sequences=3, pages=24, page=16)
    with torch.no_grad():
        want = alone(model, tokens, PROMPTS)
        positions = cache.prepare(PROMPTS)
        out = model(input_ids=padded([t[:n] for t, n in zip(tokens, PROMPTS)]), position_ids=positions.to(DEV), past_key_values=cache, use_cache=True).logits
        for b, n in enumerate(PROMPTS):
            close(out[b, :n], want[b][:n], dtype)
        assert cache.lengths() == PROMPTS and cache.get_seq_length() == max(PROMPTS)
        done = list(PROMPTS)
        for counts in ([1, 1, 1], [2, 1, 0], [1, 2, 1], [1, 1, 3]):  # single rows, several at once, and sequences that pause
            rows = [t[n:n + c] for t, n, c in zip(tokens, done, counts)]
            positions = cache.prepare(counts)
            out = model(input_ids=padded(rows), position_ids=positions.to(DEV), past_key_values=cache, use_cache=True).logits
            for b, c in enumerate(counts):
                close(out[b, :c], want[b][done[b]:done[b] + c], dtype) if c else None
                done[b] += c
        assert cache.lengths() == done == [n + steps for n in PROMPTS]
        # a sequence ends, and another begins in its row
        cache.release(1)
        positions = cache.prepare([0, 30, 0])
        out = model(input_ids=padded([[], tokens[0][:30], []]), position_ids=positions.to(DEV), past_key_values=cache, use_cache=True).logits
        close(out[1, :30], want[0][:30], dtype)


def test_equal_sequences_need_nothing_prepared_and_generate_runs():
    from transformers import DynamicCache

    model = tp.tensor_parallel(llama(torch.bfloat16), [DEV, DEV])
    tp.attention.fuse_rotary_(model, assume_no_padding=True)  # (a growing cache takes a chunk behind a prompt on the caller's word alone)
    ids = torch.randint(2, 300, (2, 50), generator=torch.Generator().manual_seed(3)).to(DEV)
    caches = [DynamicCache(), tp.paged.PagedCache(sequences=2, pages=16, page=16)]
    with torch.no_grad():
        for rows in (ids, ids[:, :1], ids[:, :7], ids[:, 3:4]):  # prompt, step, a chunk behind it, step
            want, got = (model(input_ids=rows, past_key_values=c, use_cache=True).logits for c in caches)
            close(got, want, torch.bfloat16)
        assert caches[1].lengths() == [59, 59] == [caches[0].get_seq_length()] * 2
        out = model.generate(ids, attention_mask=torch.ones_like(ids), past_key_values=tp.paged.PagedCache(sequences=2, pages=16, page=16), max_new_tokens=12, do_sample=False)
    assert out.shape == (2, 62)


def test_a_captured_step_on_pages_is_the_eager_one():
    model = tp.tensor_parallel(llama(torch.bfloat16), [DEV, DEV])
    tp.attention.fuse_rotary_(model, assume_no_padding=True)  # (transformers makes the causal mask where a forward is captured)
    g = torch.Generator().manual_seed(4)
    prompts = torch.randint(2, 300, (3, 100), generator=g).to(DEV)
    tokens = torch.randint(2, 300, (6, 3, 1), generator=g).to(DEV)
    caches = [tp.paged.PagedCache(sequences=3, pages=32, page=16) for _ in range(2)]
    with torch.no_grad():
        for cache in caches:
            model(input_ids=prompts, position_ids=cache.prepare(PROMPTS).to(DEV), past_key_values=cache, use_cache=True)
        eager, held = caches
        positions = held.prepare([1, 1, 1], hold=True).to(DEV)
        graph = tp.graphs.capture(model, input_ids=tokens[0], position_ids=positions, past_key_values=held, use_cache=True)
        for i, token in enumerate(tokens):
            counts = [1, 1, 1] if i != 3 else [1, 0, 1]
            want = model(input_ids=token, position_ids=eager.prepare(counts).to(DEV), past_key_values=eager, use_cache=True).logits
            if i:
                positions = held.prepare(counts, hold=True).to(DEV)
            got = graph(input_ids=token, position_ids=positions, past_key_values=held, use_cache=True).logits
            for b, c in enumerate(counts):
                if c:
                    close(got[b], want[b], torch.bfloat16)
            torch.cuda.synchronize()
        assert held.lengths() == eager.lengths() == [n + 6 - (b == 1) for b, n in enumerate(PROMPTS)]


def test_what_a_paged_cache_refuses():
    model = tp.tensor_parallel(llama(torch.bfloat16), [DEV])
    ids = torch.randint(2, 300, (2, 9)).to(DEV)
    with torch.no_grad():
        with pytest.raises(NotImplementedError, match="fuse_rotary_"):
            model(input_ids=ids, past_key_values=tp.paged.PagedCache(2, 8), use_cache=True)
        tp.attention.fuse_rotary_(model)
        with pytest.raises(ValueError, match="sequences"):
            model(input_ids=ids, past_key_values=tp.paged.PagedCache(3, 8), use_cache=True)
        mask = torch.ones_like(ids)
        mask[0, :3] = 0
        with pytest.raises(NotImplementedError, match="mask"):
            model(input_ids=ids, attention_mask=mask, past_key_values=tp.paged.PagedCache(2, 8), use_cache=True)
        cache = tp.paged.PagedCache(2, 8)
        cache.prepare([4, 4])
        with pytest.raises(ValueError, match="prepared"):
            model(input_ids=ids, past_key_values=cache, use_cache=True)
        cache.prepare([9, 3])
        model(input_ids=ids, past_key_values=cache, use_cache=True)
        with pytest.raises(ValueError, match="position_ids"):
            model(input_ids=ids[:, :1], past_key_values=cache, use_cache=True)
        with pytest.raises(RuntimeError, match="pages"):
            model(input_ids=torch.zeros(2, 300, dtype=torch.int64, device=DEV), position_ids=torch.zeros(2, 300, dtype=torch.int64, device=DEV), past_key_values=cache, use_cache=True)
