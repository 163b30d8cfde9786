"""Modules and decoder for many requests: what needs no GPU."""
from __future__ import annotations

import pytest
import torch

from ade_b200 import kernels, synth
from ade_b200.batch_serving import BatchDecoder, DeltaRoute, MultiDeltaLinear, attach_multi_deltas
from ade_b200.serving import LINEAR_MODULE_NAMES


def _llama(**change):
    from transformers import LlamaConfig, LlamaForCausalLM

    torch.manual_seed(0)
    cfg = LlamaConfig(**{**dict(hidden_size=128, intermediate_size=256, num_hidden_layers=2, num_attention_heads=2, vocab_size=50), **change})
    return LlamaForCausalLM(cfg).to(torch.bfloat16).eval()


def _deltas(sd, seed, skip=()):
    return {f"model.layers.{li}.{n}": synth.random_packed(*sd[f"model.layers.{li}.{n}.weight"].shape, 128, seed=seed + 10 * li + i)
            for li in range(2) for i, n in enumerate(LINEAR_MODULE_NAMES) if n not in skip}


@pytest.mark.parametrize("change", [{"attention_bias": True}, {"mlp_bias": True}, {"attention_bias": True, "mlp_bias": True}, {}], ids=str)
def test_biases_of_the_base_stay(change):
    """Rows of the base model are answered by the same operations as before: the same bits.  With the biases in the mapping and without."""
    model = _llama(**change)
    g = torch.Generator().manual_seed(1)
    with torch.no_grad():
        for n, p in model.named_parameters():
            if n.endswith(".bias"):
                p.copy_(torch.randn(p.shape, generator=g) * 0.5)
    sd = {k: v.clone() for k, v in model.state_dict().items()}
    weights = {k: v for k, v in sd.items() if not k.endswith(".bias")}
    ids = torch.arange(7)[None]
    with torch.no_grad():
        want = model(input_ids=ids).logits
        for given in (sd, weights, sd):               # the third time in place of the modules of the second
            assert attach_multi_deltas(model, given, [_deltas(sd, 1), _deltas(sd, 2, skip=LINEAR_MODULE_NAMES[1:3])], device="cpu") == 14
            assert torch.equal(model(input_ids=ids).logits, want)
        assert len([n for n, _ in model.named_buffers() if n.endswith("proj.bias")]) == sum(k.endswith(".bias") for k in sd)
        # the mapping's bias goes before the module's
        moved = {k: v + 1 if k.endswith(".bias") else v for k, v in sd.items()}
        attach_multi_deltas(model, moved, [_deltas(sd, 1)], device="cpu")
        assert torch.equal(model(input_ids=ids).logits, want) != bool(change)


def test_a_bias_of_another_size_is_refused():
    form = kernels.pack_int4(synth.random_packed(32, 128, 128, 1))
    for bias in (torch.zeros(128), torch.zeros(1), torch.zeros(32, 1)):
        with pytest.raises(ValueError, match="bias"):
            MultiDeltaLinear(torch.zeros(32, 128), [form], DeltaRoute(1), bias)


@pytest.mark.parametrize("dim", [16, 48, 80, 100, 288])
def test_head_dimensions_without_a_kernel_are_refused(dim):
    with pytest.raises(ValueError, match=f"multiple of 32 up to 256.* {dim}"):
        BatchDecoder(_llama(head_dim=dim), 2, 16)
    with pytest.raises(ValueError, match="multiple of 32"):
        BatchDecoder(_llama(hidden_size=2 * dim), 2, 16)
    with pytest.raises(ValueError, match="CUDA device"):             # the only thing wrong with this one
        BatchDecoder(_llama(head_dim=96), 2, 16)


def _hook(where, kind="register_forward_hook"):
    return lambda m: getattr(m.get_submodule(where) if where else m, kind)(lambda *a: None)


def _replace(where, change):
    """`change`d copy of the module at `where` in its place."""
    def edit(m):
        owner, _, leaf = where.rpartition(".")
        owner = m.get_submodule(owner)
        setattr(owner, leaf, change(getattr(owner, leaf)))
    return edit


def _other_forward(where):
    def edit(m):
        mod = m.get_submodule(where) if where else m
        forward = mod.forward
        mod.forward = lambda *a, **kw: forward(*a, **kw)
    return edit


def _subclass(where):
    def edit(m):
        mod = m.get_submodule(where) if where else m
        base = type(mod)
        mod.__class__ = type("Own" + base.__name__, (base,), {"forward": lambda self, *a, **kw: base.forward(self, *a, **kw)})
    return edit


class _Wrapped(torch.nn.Module):
    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, *a, **kw):
        return self.inner(*a, **kw)


PASSED_BY = ["", "model", "model.norm", "model.layers.1", "model.layers.0.self_attn", "model.layers.1.mlp", "model.layers.0.input_layernorm", "model.layers.1.post_attention_layernorm"]


@pytest.mark.parametrize("where, change", [(w, c) for w in PASSED_BY for c in (_hook(w), _hook(w, "register_forward_pre_hook"), _other_forward(w), _subclass(w))]
                         + [(w, _replace(w, _Wrapped)) for w in PASSED_BY[2:]] + [("model.layers.1.mlp", c("model.layers.1.mlp.act_fn")) for c in (_hook, _other_forward)])
@pytest.mark.parametrize("fused", ["no", "before", "behind"])
def test_modules_that_a_step_passes_by_have_to_be_the_stock_ones(where, change, fused):
    """A step does the work of these modules itself: a hook, another forward, a subclass or a wrapper in their place would act on prompts alone."""
    from ade_b200.decode_ops import enable_fused_decode_ops

    model = _llama()
    if fused == "before":
        enable_fused_decode_ops(model)
    change(model)
    if fused == "behind" and not isinstance(model.model.layers[1], _Wrapped):      # which asks every layer for its norms
        enable_fused_decode_ops(model)
    with pytest.raises(ValueError, match=f"{where or 'the model'} has") as e:
        BatchDecoder(model, 2, 16)
    assert "CUDA" not in str(e.value)


def test_hooks_for_all_modules_are_seen():
    handle = torch.nn.modules.module.register_module_forward_hook(lambda *a: None)
    try:
        with pytest.raises(ValueError, match="hooks"):
            BatchDecoder(_llama(), 2, 16)
    finally:
        handle.remove()


@pytest.mark.parametrize("change", [
    lambda m: None, lambda m: m(input_ids=torch.arange(3)[None], output_hidden_states=True), _hook("model.layers.0.self_attn.q_proj"), _hook("lm_head"), _hook("model.embed_tokens"),
    _replace("lm_head", _Wrapped), _replace("model.layers.0.mlp.up_proj", _Wrapped)])
@pytest.mark.parametrize("fused", [False, True])
def test_what_a_step_calls_may_be_anything(change, fused):
    """Nothing is wrong with these but where they are: linear modules, head and embedding are called; transformers' own hooks collect nothing."""
    from ade_b200.decode_ops import enable_fused_decode_ops

    model = _llama()
    if fused:
        enable_fused_decode_ops(model)
    change(model)
    with pytest.raises(ValueError, match="CUDA device"):
        BatchDecoder(model, 2, 16)


@pytest.mark.parametrize("where", ["model.norm", "model.layers.0.input_layernorm", "model.layers.1.post_attention_layernorm"])
@pytest.mark.parametrize("change", [torch.float32, torch.float16, "meta"])
def test_norms_of_another_type_or_device_are_refused(where, change):
    """Their launches read the weights as bfloat16 of the model's device, by their address."""
    model = _llama()
    model.get_submodule(where).to(change)
    with pytest.raises(ValueError, match=f"{where} must be in bfloat16"):
        BatchDecoder(model, 2, 16)
