"""The text encoder's checkpoint layout and refusals on the host (weights stay on the CPU, nothing is launched)."""
import json
import os

import pytest
import torch

KW = dict(vocab_size=120, d_model=128, d_kv=64, num_heads=2, d_ff=192, num_layers=2, relative_attention_num_buckets=32, relative_attention_max_distance=128,
          feed_forward_proj="gated-gelu", layer_norm_epsilon=1e-6)


def _t5(seed=0):
    transformers = pytest.importorskip("transformers")
    torch.manual_seed(seed)
    return transformers.T5EncoderModel(transformers.T5Config(**KW, dropout_rate=0.0)).eval()


def test_from_pretrained_sharded(hip_lib, tmp_path):
    from safetensors.torch import save_file
    from aether_amd.text_encoder import AetherTextEncoder
    sd = {k: v.to(torch.bfloat16).contiguous() for k, v in _t5().state_dict().items() if k != "encoder.embed_tokens.weight"}
    root = tmp_path / "text_encoder"
    os.makedirs(root)
    json.dump(dict(KW, model_type="t5", architectures=["T5EncoderModel"]), open(root / "config.json", "w"))
    keys = sorted(sd)
    weight_map = {}
    for i in range(2):
        part = {k: sd[k].clone() for k in keys[i::2]}
        save_file(part, str(root / f"model-{i + 1:05d}-of-00002.safetensors"))
        weight_map.update({k: f"model-{i + 1:05d}-of-00002.safetensors" for k in part})
    json.dump({"weight_map": weight_map}, open(root / "model.safetensors.index.json", "w"))
    m = AetherTextEncoder.from_pretrained(str(tmp_path), device="cpu")
    att, ff = "encoder.block.1.layer.0.SelfAttention.", "encoder.block.1.layer.1.DenseReluDense."
    assert torch.equal(m.embedding, sd["shared.weight"]) and torch.equal(m.bias_table, sd["encoder.block.0.layer.0.SelfAttention.relative_attention_bias.weight"])
    b = m.blocks[1]
    assert torch.equal(b.qkv[128:256], sd[att + "k.weight"]) and torch.equal(b.out, sd[att + "o.weight"])
    assert torch.equal(b.gate, sd[ff + "wi_0.weight"]) and torch.equal(b.up, sd[ff + "wi_1.weight"]) and torch.equal(b.down, sd[ff + "wo.weight"])
    assert b.norm2.dtype == torch.float32 and torch.equal(b.norm2, sd["encoder.block.1.layer.1.layer_norm.weight"].float())
    assert sum(p.numel() for p in m.parameters()) == sum(v.numel() for v in sd.values()) and not any(p.requires_grad for p in m.parameters())
    assert next(m.parameters()).device.type == "cpu"
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        m(torch.zeros(1, 4, dtype=torch.int64))
    with pytest.raises(ValueError, match="bfloat16"):
        AetherTextEncoder.from_pretrained(str(tmp_path), device="cpu", torch_dtype=torch.float32)
    bad = dict(sd)
    bad[att + "k.weight"] = bad[att + "k.weight"][:64]
    with pytest.raises(ValueError, match="rows"):
        m.load_t5_state_dict(bad)


@pytest.mark.parametrize("kw", [dict(feed_forward_proj="relu"), dict(d_kv=32), dict(d_model=100), dict(d_ff=100), dict(relative_attention_num_buckets=7),
                                dict(relative_attention_max_distance=8), dict(relative_attention_max_distance=100000), dict(d_model=32768)])
def test_unsupported_configurations(hip_lib, kw):
    from aether_amd.text_encoder import AetherTextEncoder
    with pytest.raises(ValueError):
        AetherTextEncoder({**KW, "num_layers": 0, **kw}, device="meta")


def test_demo_flag():
    import importlib
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "scripts"))
    demo = importlib.import_module("demo")
    args = demo.parse_args(["--task", "prediction"])
    assert args.native_text_encoder is False
    assert demo.parse_args(["--task", "prediction", "--native_text_encoder"]).native_text_encoder is True


def test_loading_drops_the_eight_bit_copies(hip_lib):
    """New weights by this module's own load_state_dict, or by that of a module around it: 8-bit copies of the old ones do not stay."""
    import torch
    from aether_amd.text_encoder import AetherTextEncoder
    m = AetherTextEncoder(dict(vocab_size=32, d_model=128, num_heads=2, d_ff=128, num_layers=1), device="cpu")
    outer = torch.nn.ModuleDict({"text": m})
    for load in (lambda: m.load_state_dict(m.state_dict()), lambda: outer.load_state_dict(outer.state_dict()), lambda: outer.to(torch.device("cpu"))):
        m._e4m3 = [()]
        load()
        assert m._e4m3 is None


def test_dropped_eight_bit_copies_are_named(hip_lib):
    """Where 8-bit weights go, a warning says that the 16-bit ones serve from there; nothing is said where there were none."""
    import warnings
    from aether_amd.text_encoder import AetherTextEncoder
    m = AetherTextEncoder(dict(vocab_size=32, d_model=128, num_heads=2, d_ff=128, num_layers=1), device="cpu")
    sd = {"shared.weight": m.embedding, "encoder.block.0.layer.0.SelfAttention.relative_attention_bias.weight": m.bias_table, "encoder.final_layer_norm.weight": m.final_norm}
    b, inner = m.blocks[0], 128
    sd.update({f"encoder.block.0.layer.0.SelfAttention.{n}.weight": b.qkv[i * inner:(i + 1) * inner] for i, n in enumerate("qkv")})
    sd.update({"encoder.block.0.layer.0.SelfAttention.o.weight": b.out, "encoder.block.0.layer.0.layer_norm.weight": b.norm1, "encoder.block.0.layer.1.layer_norm.weight": b.norm2,
               "encoder.block.0.layer.1.DenseReluDense.wi_0.weight": b.gate, "encoder.block.0.layer.1.DenseReluDense.wi_1.weight": b.up,
               "encoder.block.0.layer.1.DenseReluDense.wo.weight": b.down})
    sd = {k: v.detach().clone() for k, v in sd.items()}
    for drop in (lambda: m.to("cpu"), lambda: m.load_state_dict(m.state_dict()), lambda: m.load_t5_state_dict(sd), lambda: m.init_random_weights()):
        m._e4m3 = [()]
        with pytest.warns(UserWarning, match="quantize_feed_forward"):
            drop()
        assert m._e4m3 is None
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            drop()
    m._e4m3 = [()]
    with pytest.warns(UserWarning), pytest.raises(KeyError):
        m.load_t5_state_dict({k: v for k, v in sd.items() if "final" not in k})
    assert m._e4m3 is None
