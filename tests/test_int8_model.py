"""A checkpoint in 8-bit integers through the loader and the decoder: what is accepted, where its tensors go, and the model's steps
against the operators one behind the other (each of which has its own tests against 64 bits)."""

from __future__ import annotations

import copy
import dataclasses
import json

import pytest
import torch

from tandem_amd import decode_graph, loader, model as tmodel
from tandem_amd.kv_cache import PagedKVCache
from tandem_amd.layers import norm, w8

CFG = tmodel.DecoderConfig(hidden_size=512, intermediate_size=1040, num_heads=4, num_kv_heads=2, head_dim=128, num_layers=2,
                           vocab_size=777, qk_norm=True, rope_theta=1e4)
ARGS = {"num_bits": 8, "type": "int", "symmetric": True}
CONFIG = {"quant_method": "compressed-tensors", "format": "int-quantized", "quantization_status": "compressed", "ignore": ["lm_head"],
          "kv_cache_scheme": None, "config_groups": {"group_0": {
              "targets": ["Linear"], "output_activations": None,
              "weights": {**ARGS, "strategy": "channel", "dynamic": False, "group_size": None, "actorder": None},
              "input_activations": {**ARGS, "strategy": "token", "dynamic": True}}}}


def test_config():
    assert loader.QuantConfig.from_dict(CONFIG) == loader.QuantConfig("compressed-tensors", 8, 0)

    def changed(*path_value):
        d = copy.deepcopy(CONFIG)
        *path, last, value = path_value
        at = d
        for p in path:
            at = at[p]
        at[last] = value
        return d

    group = ("config_groups", "group_0")
    for bad, needle in ((changed("format", "pack-quantized"), "pack-quantized"), (changed("ignore", []), "lm_head"),
                        (changed("ignore", ["lm_head", "model.layers.0.mlp.down_proj"]), "ignore"), (changed("kv_cache_scheme", {"num_bits": 8}), "kv_cache"),
                        (changed("config_groups", {}), "config_groups"), (changed("config_groups", {**CONFIG["config_groups"], "group_1": {}}), "config_groups"),
                        (changed(*group, "targets", ["re:.*mlp.*"]), "targets"), (changed(*group, "input_activations", None), "input_activations"),
                        (changed(*group, "weights", "num_bits", 4), "num_bits"), (changed(*group, "weights", "type", "float"), "type"),
                        (changed(*group, "weights", "symmetric", False), "symmetric"), (changed(*group, "weights", "strategy", "group"), "strategy"),
                        (changed(*group, "weights", "actorder", "static"), "actorder"), (changed(*group, "input_activations", "dynamic", False), "dynamic"),
                        (changed(*group, "input_activations", "strategy", "tensor"), "strategy"), (changed(*group, "output_activations", ARGS), "output_activations"),
                        (changed("quantization_status", "frozen"), "frozen"), (changed("sparsity_config", {"format": "sparse-24-bitmask"}), "sparsity"),
                        (changed("transform_config", {"config_groups": {"u": {}}}), "transform")):
        with pytest.raises(NotImplementedError, match=needle):
            loader.QuantConfig.from_dict(bad)


def _checkpoint(path, cfg=CFG, seed=0) -> dict[str, torch.Tensor]:
    from safetensors.torch import save_file

    g = torch.Generator().manual_seed(seed)
    h, i, d = cfg.hidden_size, cfg.intermediate_size, cfg.head_dim
    q, kv = cfg.num_heads * d, cfg.num_kv_heads * d
    t = {"model.embed_tokens.weight": torch.randn(cfg.vocab_size, h, generator=g).half(), "model.norm.weight": torch.rand(h, generator=g).half() + 0.5,
         "lm_head.weight": (torch.randn(cfg.vocab_size, h, generator=g) * 0.05).half()}
    for n in range(cfg.num_layers):
        at = f"model.layers.{n}."
        for name, rows, width in (("self_attn.q_proj", q, h), ("self_attn.k_proj", kv, h), ("self_attn.v_proj", kv, h), ("self_attn.o_proj", h, q),
                                  ("mlp.gate_proj", i, h), ("mlp.up_proj", i, h), ("mlp.down_proj", h, i)):
            t[at + name + ".weight"] = torch.randint(-127, 128, (rows, width), generator=g, dtype=torch.int8)
            t[at + name + ".weight_scale"] = ((0.5 + torch.rand(rows, 1, generator=g)) * width ** -0.5 / 60).bfloat16()
        for name, width in (("input_layernorm", h), ("post_attention_layernorm", h), ("self_attn.q_norm", d), ("self_attn.k_norm", d)):
            t[at + name + ".weight"] = torch.rand(width, generator=g).half() + 0.5
    save_file(t, str(path / "model.safetensors"))
    (path / "config.json").write_text(json.dumps({"quantization_config": CONFIG}))
    return t


def _load(path):
    quant = loader.QuantConfig.from_dict(json.loads((path / "config.json").read_text())["quantization_config"])
    model = tmodel.DecoderModel(CFG, quant)
    loader.load_weights(model, str(path))
    return model


def test_tensors_go_where_they_belong(tmp_path):
    t = _checkpoint(tmp_path)
    model = _load(tmp_path)
    for n, layer in enumerate(model.model.layers):
        for mod, at, parts in ((layer.self_attn.qkv_proj, "self_attn", ("q_proj", "k_proj", "v_proj")), (layer.self_attn.o_proj, "self_attn", ("o_proj",)),
                               (layer.mlp.gate_up_proj, "mlp", ("gate_proj", "up_proj")), (layer.mlp.down_proj, "mlp", ("down_proj",))):
            assert isinstance(mod, w8.W8Linear) and mod.silu_mul is (parts[0] == "gate_proj")
            names = [f"model.layers.{n}.{at}.{p}" for p in parts]
            assert torch.equal(mod.weight, torch.cat([t[x + ".weight"] for x in names]))
            assert mod.weight_scale.dtype == torch.float32 and torch.equal(mod.weight_scale, torch.cat([t[x + ".weight_scale"] for x in names]).float())
    from safetensors.torch import save_file

    t["model.layers.0.mlp.down_proj.weight"] = t["model.layers.0.mlp.down_proj.weight"].half()
    save_file(t, str(tmp_path / "model.safetensors"))
    with pytest.raises(ValueError, match="int8"):
        _load(tmp_path)


def test_random_weights():
    model = tmodel.init_random(tmodel.DecoderModel(dataclasses.replace(CFG, num_layers=1), loader.QuantConfig.from_dict(CONFIG)), seed=1)
    mod = model.model.layers[0].mlp.down_proj
    w = mod.weight.float() * mod.weight_scale
    assert abs(float(w.std()) / 0.02 - 1) < 0.05 and int(mod.weight.abs().max()) <= 127


def _by_operators(model, ids):
    """The one-token step from the public operators."""
    hidden, residual = model.model.embed_tokens.weight[ids], None
    group = CFG.num_heads // CFG.num_kv_heads

    def product(mod, codes, scales):
        return w8.linear_int8(codes, scales, mod.weight, mod.weight_scale, silu_mul=mod.silu_mul)

    for layer in model.model.layers:
        n1, n2 = layer.input_layernorm, layer.post_attention_layernorm
        if residual is None:
            residual = hidden.clone()
            codes, scales = norm.rms_norm_int8(hidden, n1.weight, n1.eps)
        else:
            codes, scales, residual = norm.fused_add_rms_norm_int8(hidden, residual, n1.weight, n1.eps)
        v = product(layer.self_attn.qkv_proj, codes, scales)[:, -CFG.num_kv_heads * 128:].view(-1, CFG.num_kv_heads, 1, 128)
        attended = v.expand(-1, -1, group, -1).reshape(len(ids), -1)
        hidden = product(layer.self_attn.o_proj, *w8.quantize_int8(attended))
        codes, scales, residual = norm.fused_add_rms_norm_int8(hidden, residual, n2.weight, n2.eps)
        hidden = product(layer.mlp.down_proj, *w8.quantize_int8(product(layer.mlp.gate_up_proj, codes, scales)))
    n = model.model.norm
    return norm.fused_add_rms_norm(hidden, residual, n.weight, n.eps)[0]


@pytest.mark.gpu
def test_steps(tmp_path):
    """Eager, bit for bit the operators; the captured step over a paged cache, bit for bit the eager one over another cache, behind
    prompts of their own; and the codes' effect on the result against the dequantised weights and unquantised activations."""
    _checkpoint(tmp_path)
    device = torch.device("cuda", 0)
    model = tmodel.prepare(_load(tmp_path), device)
    with torch.inference_mode():
        for m in (1, 5, 40, 130):
            ids = torch.arange(m, device=device) * 5 % CFG.vocab_size
            assert torch.equal(model(ids), _by_operators(model, ids))

        prompts = [[5, 9, 700, 3, 3, 8, 1], [11], [2] * 33]
        caches = [PagedKVCache.for_model(CFG, 32, 4, 128, device=device) for _ in range(2)]
        ids = torch.tensor([i for p in prompts for i in p], device=device)
        lens = torch.tensor([len(p) for p in prompts] + [0], dtype=torch.int32, device=device)
        firsts = [model(ids, c.plan(lens, len(ids))) for c in caches]
        assert torch.equal(*firsts)
        runner = decode_graph.DecodeGraphRunner(model, 4, device, cache=caches[0])
        one = torch.tensor([1, 1, 1, 0], dtype=torch.int32, device=device)
        for step in range(6):
            ids = [7 + step, 400 - step, 70 * step]
            got = runner.run(ids + [-1]).clone()
            want = model.compute_logits(model(torch.tensor(ids, device=device), caches[1].plan(one, 3, max_query_len=1)))
            assert torch.equal(got, want), step


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 7, 50, 200])
def test_mlp_against_real_numbers(m):
    """norm, gate_up, SwiGLU, down against the same block without any quantisation of activations, in 64 bits. A code is off by half a step
    of its row's scale, uniformly: sigma 1 / sqrt(12) steps. Output = sum of K independent errors times weights, so that its error has the size
    of scale / sqrt(12) |w row|, once through down and once, scaled by the block's slope, through gate_up. That is checked as a ratio of
    norms: N(0, 1) rows of 512 to 1040 values have maxima of 3 to 5 sigma, so an error of 5 / 127 / sqrt(12) = 0.0114 of the values at most
    for each of the two stages (gate and up: two of the first), and 0.0114 (1 + 2 * 1.2) < 0.04 in all."""
    g = torch.Generator(device="cuda").manual_seed(m)
    mlp = tmodel.GatedMLP(512, 1040, loader.QuantConfig("compressed-tensors", 8, 0)).cuda()
    for mod in (mlp.gate_up_proj, mlp.down_proj):
        mod.weight.copy_(torch.randint(-127, 128, mod.weight.shape, device="cuda", dtype=torch.int8, generator=g))
        mod.weight_scale.copy_((0.5 + torch.rand(mod.weight_scale.shape, device="cuda", generator=g)) * mod.in_features ** -0.5 / 73)
    x = torch.randn(m, 512, device="cuda", generator=g).half()
    r = torch.randn(m, 512, device="cuda", generator=g).half()
    weight = (0.5 + torch.rand(512, device="cuda", generator=g)).half()
    s = x.double() + r.double()
    y, out = mlp.gate_up_proj.forward_norm(x, r, weight, 1e-6)
    y = mlp.down_proj(y)
    a = s * torch.rsqrt((s * s).mean(-1, keepdim=True) + 1e-6) * weight.double()
    gate, up = (a @ (mlp.gate_up_proj.weight.double() * mlp.gate_up_proj.weight_scale.double()).t()).chunk(2, dim=1)
    want = (gate * torch.sigmoid(gate) * up) @ (mlp.down_proj.weight.double() * mlp.down_proj.weight_scale.double()).t()
    assert float((y.double() - want).norm() / want.norm()) < 0.04 and torch.equal(out, s.half())
