"""Models of 8-bit rows on the device: what they leave of their 16-bit weights, and what moving and reloading them leaves of the layout that their products are fastest on."""
import weakref

import pytest
import torch

import tensor_parallel_amd as tp
from tensor_parallel_amd import int8, shard_modules
from tensor_parallel_amd.int8 import quantize_linears_

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def llama(hidden=528):
    from transformers import LlamaConfig, LlamaForCausalLM

    torch.manual_seed(0)
    config = LlamaConfig(vocab_size=300, hidden_size=hidden, intermediate_size=720, num_hidden_layers=1, num_attention_heads=6, num_key_value_heads=2, head_dim=64, max_position_embeddings=256)
    model = LlamaForCausalLM(config).to(DEV, torch.bfloat16).eval()
    model.config._attn_implementation = tp.attention.register()
    shard_modules.install_shard_kernels(model)
    tp.attention.fuse_rotary_(model)
    return model


@pytest.mark.parametrize("activations", [True, False])
def test_16_bit_weights_of_q_k_and_v_are_given_back(activations):
    model = llama()
    attn = model.model.layers[0].self_attn
    whole = weakref.ref(attn.__dict__["_tp_qkv"][0])
    before = torch.cuda.memory_allocated(DEV)
    bits16 = whole().numel() * 2
    n = quantize_linears_(model.model.layers, activations=activations)
    assert n == 7 and whole() is None and "_tp_qkv" not in attn.__dict__
    assert before - torch.cuda.memory_allocated(DEV) > bits16 // 3  # (the codes take half, and their rows begin on 128-byte boundaries)


def test_a_model_that_moves_to_the_host_and_back():
    """Nothing of it stays on the device meanwhile; its rows begin on 128-byte boundaries again, and its logits are the same."""
    from transformers import DynamicCache

    before = torch.cuda.memory_allocated(DEV)
    model = llama()
    attn = model.model.layers[0].self_attn
    quantize_linears_(model.model.layers, activations=True)
    ids = torch.randint(2, 300, (2, 17), device=DEV)

    def forward():
        with torch.no_grad():
            return model(input_ids=ids, past_key_values=DynamicCache(), use_cache=True).logits

    want = forward()
    model.to("cpu")
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated(DEV) - before <= want.numel() * 2 + ids.numel() * 8 + 4096
    model.to(DEV)
    assert attn.q_proj.wq.stride() == (640, 1) and model.model.layers[0].mlp.down_proj.wq.stride() == (768, 1)
    assert torch.equal(forward(), want)
    tp.attention.fuse_rotary_(model)
    assert attn.q_proj.wq.untyped_storage().data_ptr() == attn.v_proj.wq.untyped_storage().data_ptr() and torch.equal(forward(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [512, 1000, 2048, 2056, 4096, 5504, 8192, 11008, 16384])
def test_a_row_has_the_same_scale_in_every_batch(d, dtype):
    """Few rows are held by more wavefronts than the many of a large launch (2^23 values): codes and scales are the same bits, and with the addition in the same launch too."""
    rows = (1 << 23) // d + 1
    g = torch.Generator(device=DEV).manual_seed(d)
    x = (torch.randn(rows, d, device=DEV, generator=g) * (torch.rand(rows, 1, device=DEV, generator=g) + 0.01)).to(dtype)
    w = (1 + 0.3 * torch.randn(d, device=DEV, generator=g)).to(dtype)
    whole = int8.rms_norm(x, w, 1e-5)
    for n in (1, 7, rows - 1):
        part = int8.rms_norm(x[:n], w, 1e-5)
        assert torch.equal(part.codes, whole.codes[:n]) and torch.equal(part.scale, whole.scale[:n])
    total, rows_ = int8.add_rms_norm(torch.zeros_like(x), x, w, 1e-5)
    assert torch.equal(total, x) and torch.equal(rows_.codes, whole.codes) and torch.equal(rows_.scale, whole.scale)
