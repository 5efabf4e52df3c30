"""An RW8 (8-bit) Llama through the engine: checkpoint, load, generate; resident, streamed and from
layer shards give the same tokens; the 8-bit layer forward is its kernels in order."""
import pytest
import torch

from rocketllm_b200 import kernels
from rocketllm_b200.engine import AutoModel, RocketModel, footprint
from rocketllm_b200.quant import Int8Rows, RW8Linear
from rocketllm_b200.quant.convert import save_rw8_checkpoint

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dense():
    from transformers import LlamaConfig, LlamaForCausalLM
    cfg = LlamaConfig(hidden_size=512, intermediate_size=1536, num_hidden_layers=3,
                      num_attention_heads=8, num_key_value_heads=2, vocab_size=2048,
                      max_position_embeddings=512, tie_word_embeddings=False)
    torch.manual_seed(0)
    model = LlamaForCausalLM(cfg)
    with torch.no_grad():
        for n, p in model.named_parameters():
            p.copy_(torch.ones_like(p) if "norm" in n else torch.randn_like(p) * 0.04)
    return model.to(torch.bfloat16).eval()


@pytest.fixture(scope="module")
def checkpoint(dense, tmp_path_factory):
    return save_rw8_checkpoint(dense, str(tmp_path_factory.mktemp("rw8")), device="cuda")


def prompt(n, batch=1):
    return torch.randint(0, 2048, (batch, n), generator=torch.Generator().manual_seed(n)).cuda()


def test_checkpoint_holds_the_quantized_weights(dense, checkpoint):
    model = AutoModel.from_pretrained(checkpoint).model
    for name, want in dense.named_modules():
        if isinstance(want, torch.nn.Linear):
            got = model.get_submodule(name)
            assert isinstance(got, RW8Linear)
            codes, scale = kernels.int8_quantize(want.weight.detach().cuda())
            assert torch.equal(got.weight, codes)
            assert torch.equal(got.weight_scale, scale[:, None])


def test_linear_module(cuda):
    torch.manual_seed(3)
    dense = torch.nn.Linear(256, 96, bias=True).to(cuda, torch.bfloat16)
    m = RW8Linear.from_linear(dense)
    m.weight.data, s = kernels.int8_quantize(dense.weight.detach())
    m.weight_scale.data = s[:, None]
    m.bias.data = dense.bias.detach()
    x = torch.randn(2, 5, 256, device=cuda).bfloat16()
    codes, scale = kernels.int8_quantize(x)
    want = kernels.int8_linear(codes, scale, m.weight, m.weight_scale, bias=m.bias)
    assert torch.equal(m(x), want)
    rows = Int8Rows(codes, scale, torch.bfloat16)
    assert torch.equal(m(rows), want) and rows.shape == x.shape and rows.device == x.device
    assert torch.equal(rows.dequantize(), kernels.int8_dequantize(codes, scale))
    res = torch.randn(2, 5, 96, device=cuda).bfloat16()
    assert torch.equal(m(rows, residual=res),
                       kernels.int8_linear(codes, scale, m.weight, m.weight_scale, bias=m.bias,
                                           residual=res))
    y = m(x.float())   # other types: the bias follows
    assert y.dtype == torch.float32


@pytest.mark.parametrize("batch,n", [(1, 1), (1, 37), (3, 130)])
def test_layer_forward_is_its_kernels_in_order(checkpoint, batch, n):
    model = AutoModel.from_pretrained(checkpoint).model
    layer = model.model.layers[1]
    seen = {}

    def keep(name):
        def hook(module, args, kwargs, out):
            seen[name] = out[0] if isinstance(out, tuple) else out
        return hook

    handles = [layer.self_attn.register_forward_hook(keep("attn"), with_kwargs=True),
               layer.register_forward_hook(keep("layer"), with_kwargs=True),
               model.model.layers[0].register_forward_hook(keep("in"), with_kwargs=True)]
    with torch.no_grad():
        model(prompt(n, batch))
    for h in handles:
        h.remove()
    codes, scale, h = kernels.int8_rmsnorm(seen["attn"], layer.post_attention_layernorm.weight,
                                           layer.post_attention_layernorm.variance_epsilon,
                                           residual=seen["in"])
    m = layer.mlp
    gate, up = (kernels.int8_linear(codes, scale, p.weight, p.weight_scale)
                for p in (m.gate_proj, m.up_proj))
    codes, scale = kernels.int8_quantize(up, gate=gate)
    want = kernels.int8_linear(codes, scale, m.down_proj.weight, m.down_proj.weight_scale,
                               residual=h)
    assert torch.equal(seen["layer"], want)


def test_logits_stay_near_the_dense_model(dense, checkpoint):
    """Half an 8-bit step against a row's root mean square is at most 0.5 * 5 / 127 / sqrt(3) =
    1.1% for rows whose largest value is below 5 root mean squares, for activations and weights
    each: 1.6% a projection.  22 projections' errors, added as independent ones, are below 8%;
    the bound is twice that."""
    ids = prompt(64)
    model = AutoModel.from_pretrained(checkpoint)
    with torch.no_grad():
        got = model(ids).logits.double()
        want = dense.to("cuda")(ids).logits.double()
    assert (got - want).norm() <= 0.16 * want.norm()


def test_streamed_and_sharded_equal_resident(checkpoint, tmp_path):
    from rocketllm_b200.shards import split_rw4_layers
    ids = prompt(16)
    resident = AutoModel.from_pretrained(checkpoint)
    rest, layers = footprint(resident.model)
    assert resident.streamer is None
    with torch.no_grad():
        logits = resident(ids).logits
        tokens = resident.generate(ids, max_new_tokens=8, do_sample=False, min_new_tokens=8)
    assert tokens.shape == (1, 24)
    streamed = RocketModel(checkpoint, vram_budget=rest + 2 * max(layers) + 1000, kv_cache="fp16")
    assert streamed.streamer is not None and streamed.streamer.window == 2
    split_rw4_layers(AutoModel.from_pretrained(checkpoint).model.cpu(), str(tmp_path / "shards"))
    sharded = RocketModel(str(tmp_path / "shards"))
    for other in (streamed, sharded):
        with torch.no_grad():
            assert torch.equal(other(ids).logits, logits)
            assert torch.equal(other.generate(ids, max_new_tokens=8, do_sample=False,
                                              min_new_tokens=8), tokens)
        other.close()


def test_int4_kv_cache_and_batches(checkpoint):
    """The 8-bit weights beside the int4 KV cache, and a left-padded batch."""
    model = RocketModel(checkpoint, kv_cache="int4")
    out = model.generate(prompt(200), max_new_tokens=4, do_sample=False)
    assert out.shape == (1, 204)
    model = AutoModel.from_pretrained(checkpoint)
    ids = prompt(20, 2)
    mask = torch.ones_like(ids)
    mask[0, :7] = 0
    with torch.no_grad():
        both = model(ids, attention_mask=mask).logits
        alone = model(ids[1:]).logits
    # a row's 8-bit products do not depend on the batch; the library's attention may round
    # otherwise, which moves a code by a step where it sits at a border: the bound above
    assert (both[1] - alone[0]).double().norm() <= 0.16 * alone.double().norm()
    out = model.generate(ids, attention_mask=mask, max_new_tokens=4, do_sample=False,
                         pad_token_id=0)
    assert out.shape == (2, 24)


@pytest.mark.parametrize("batch", [1, 3])
def test_graphed_decode(checkpoint, batch):
    """The CUDA-graphed decode step over RW8 layers: the same tokens as the same step launched
    eagerly, in a graph that stays alive beside a second one."""
    from rocketllm_b200.decode import GraphedDecoder
    model = AutoModel.from_pretrained(checkpoint).model
    ids = prompt(12, batch)
    eager = GraphedDecoder(model, batch, 64, use_graph=False).generate(ids, 16)
    decoders = [GraphedDecoder(model, batch, 64) for _ in range(2)]
    got = [d.generate(ids, 16) for d in decoders]
    assert torch.equal(got[0], eager) and torch.equal(got[1], eager)
