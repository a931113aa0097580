"""Which mixtures of experts the surgery takes: those whose function a router, its experts' three projections and SiLU.mul are.  Everything
else in a block would be left out of the replacement without a word, so it is refused."""
from types import SimpleNamespace

import pytest
import torch
import torch.nn.functional as F
from torch import nn

from sparseflow_b200.nn import replace_llama_mlp_module
from sparseflow_b200.nn.sparseflow_moe import is_moe, make_sparseflow_moe


def _expert(**kw):
    m = nn.Module()
    for name in ("gate_proj", "up_proj", "down_proj"):
        setattr(m, name, nn.Linear(64, 64, bias=False))
    for name, v in kw.items():
        setattr(m, name, v() if isinstance(v, type) else v)
    return m


def _block(expert=None, **kw):
    m = nn.Module()
    m.gate, m.experts, m.top_k = nn.Linear(64, 2, bias=False), nn.ModuleList([_expert(**(expert or {})) for _ in range(2)]), 1
    for name, v in kw.items():
        setattr(m, name, v)
    return m


def _accepted(block):
    with pytest.raises(ValueError, match="CUDA"):      # past the layout: what is refused is that the weights are not on a GPU
        make_sparseflow_moe(block)


def _refused(block, match):
    with pytest.raises(RuntimeError, match=match):
        make_sparseflow_moe(block)


def test_plain_block():
    _accepted(_block())


def test_parameters_inside_an_expert():
    _refused(_block(expert={"ln": nn.LayerNorm(64)}), "ln.weight")
    biased = _block()
    biased.experts[1].scale = nn.Parameter(biased.gate.weight[0, :1].clone())
    _refused(biased, "experts.1.scale")


def test_buffers():
    shifted = _block()
    shifted.register_buffer("e_score_correction_bias", shifted.gate.weight.detach()[:, 0].clone())
    _refused(shifted, "e_score_correction_bias")
    shifted = _block()
    shifted.register_buffer("shift", shifted.gate.weight.detach()[:, 0].clone(), persistent=False)
    _refused(shifted, "shift")
    scaled = _block()
    scaled.experts[0].register_buffer("scale", scaled.gate.weight.detach()[0, :1].clone())
    _refused(scaled, "experts.0.scale")


class _SwishWithASlope(nn.Module):
    def forward(self, x):
        return x * (1.702 * x).sigmoid()


@pytest.mark.parametrize("act", [nn.Hardswish(), F.hardswish, _SwishWithASlope(), nn.GELU(), F.gelu])
def test_relatives_of_silu(act):
    _refused(_block(expert={"act_fn": act}), "SiLU")


class SiLUActivation(nn.Module):
    def forward(self, x):
        return F.silu(x)


@pytest.mark.parametrize("act", [nn.SiLU(), nn.SiLU(inplace=True), F.silu, SiLUActivation()])
def test_silu_itself(act):
    _accepted(_block(expert={"act_fn": act}))


@pytest.mark.parametrize("name", ["act", "activation", "activation_fn", "hidden_act", "nonlinearity"])
def test_activations_under_other_names(name):
    for act in (nn.GELU(), nn.functional.relu, lambda x: x):
        _refused(_block(expert={name: act}), f"{name}.*SiLU")
    for act in (nn.SiLU(), F.silu):
        _accepted(_block(expert={name: act}))


def test_activations_by_name():
    for name in ("hidden_act", "activation", "act"):
        _refused(_block(expert={name: "gelu"}), f"{name}.*SiLU")
        _accepted(_block(expert={name: "silu"}))


def test_what_an_expert_does_beside_its_products():
    _refused(_block(expert={"norm": nn.LayerNorm(64, elementwise_affine=False)}), "norm")
    patched = _block()
    patched.experts[1].forward = lambda x: 2 * x
    _refused(patched, "forward")
    _accepted(_block(expert={"drop": nn.Dropout(0.1), "nothing": nn.Identity()}))


@pytest.mark.parametrize("setting", [{"routed_scaling_factor": 2.5}, {"router_scale": 0.5}, {"scoring_func": "sigmoid"}, {"score_function": "sigmoid"},
                                     {"n_group": 8}, {"topk_group": 4}, {"topk_method": "noaux_tc"}, {"router_softcapping": 30.0}])
def test_other_routing(setting):
    (name, _), = setting.items()
    _refused(_block(**setting), name)
    if name not in ("router_scale", "router_softcapping"):
        _refused(_block(config=SimpleNamespace(**setting)), name)


def test_functions_of_the_block():
    _refused(_block(score=torch.sigmoid), "score")
    _refused(_block(post=nn.LayerNorm(64, elementwise_affine=False)), "post")
    _accepted(_block(score=torch.softmax, other=F.softmax, third=nn.Softmax(-1), drop=nn.Dropout(0.1)))


def test_settings_that_change_nothing():
    _accepted(_block(routed_scaling_factor=1.0, scoring_func="softmax", n_group=1, topk_group=None, topk_method="greedy", norm_topk_prob=False,
                     num_experts=2, hidden_dim=64, hidden_act="silu", jitter_noise=0.1, config=SimpleNamespace(rope_scaling_factor=8.0, n_group=1)))


def _model(mlp):
    model, layer = nn.Module(), nn.Module()
    layer.mlp = mlp
    model.layers = nn.ModuleList([layer])
    return model


@pytest.mark.parametrize("experts", [8, None, nn.Linear(64, 64), nn.ModuleList(), nn.ModuleDict({"a": nn.Linear(64, 64)}), [1, 2]])
def test_experts_that_are_no_list(experts):
    """Not a mixture that is read, and no other error than for every layout that the surgery does not know."""
    m = nn.Module()
    m.gate, m.experts = nn.Linear(64, 2, bias=False), experts
    assert not is_moe(m)
    for call in (lambda: make_sparseflow_moe(m), lambda: replace_llama_mlp_module(_model(m), None)):
        with pytest.raises(RuntimeError, match="Unsupported"):
            call()


def test_down_mode():
    """"dense", the default, promises an unpruned down projection: a mixture keeps it only where pruning changes nothing."""
    with pytest.raises(RuntimeError, match="down_mode"):
        replace_llama_mlp_module(_model(_block()), None)
    with pytest.raises(RuntimeError, match="down_mode"):
        replace_llama_mlp_module(_model(_block()), None, down_mode="dense")
    with pytest.raises(ValueError, match="down_mode"):
        replace_llama_mlp_module(_model(_block()), None, down_mode="half")
    with pytest.raises(ValueError, match="CUDA"):
        replace_llama_mlp_module(_model(_block()), None, down_mode="sparse")
    pruned = _block()
    for e in pruned.experts:
        e.down_proj.weight.data[:, 1::4] = 0
        e.down_proj.weight.data[:, 2::4] = 0
    with pytest.raises(ValueError, match="CUDA"):
        replace_llama_mlp_module(_model(pruned), None)
    pruned.experts[1].down_proj.weight.data[5, 9] = 0.5      # one group of four with three values
    with pytest.raises(RuntimeError, match="down_mode"):
        replace_llama_mlp_module(_model(pruned), None)


class _AdaptedLinear(nn.Linear):
    def __init__(self, *args):
        super().__init__(*args, bias=False)
        self.lora_a, self.lora_b = nn.Linear(64, 4, bias=False), nn.Linear(4, 64, bias=False)

    def forward(self, x):
        return super().forward(x) + self.lora_b(self.lora_a(x))


def test_projections_that_do_more_or_are_something_else():
    _refused(_block(expert={"down_proj": _AdaptedLinear(64, 64)}), "lora_a")
    routed = _block()
    routed.gate.extra = nn.Parameter(routed.gate.weight.detach().clone())
    _refused(routed, "gate.extra")
    other = nn.Module()
    other.weight = nn.Parameter(routed.gate.weight.detach().clone())
    _refused(_block(expert={"up_proj": other}), "nn.Linear")


def test_experts_in_a_plain_list():
    """Not registered with the block: looked through all the same."""
    def block(**kw):
        m = _block()
        experts = [_expert(**kw) for _ in range(2)]
        del m.experts
        m.experts = experts
        return m

    _accepted(block())
    _refused(block(ln=nn.LayerNorm(64)), "ln.weight")
    scaled = block()
    scaled.experts[0].register_buffer("scale", scaled.gate.weight.detach()[0, :1].clone())
    _refused(scaled, "scale")
    _refused(block(act_fn=nn.GELU()), "SiLU")


@pytest.mark.parametrize("setting", [{"alpha": 1.702}, {"swiglu_limit": 7.0}, {"output_multiplier": 0.5}, {"clamp_value": 10}])
def test_settings_of_an_expert(setting):
    (name, _), = setting.items()
    _refused(_block(expert=setting), name)
    _refused(_block(**setting), name)
    _accepted(_block(expert={name: None, "hidden_size": 64, "intermediate_size": 64, "config": SimpleNamespace(alpha=2.0)}))


def test_bounds_on_the_tokens_of_an_expert():
    _refused(_block(capacity_factor=1.25), "capacity_factor")
    _accepted(_block(capacity_factor=None))


def test_normalisation_of_the_weights(monkeypatch):
    made = []
    monkeypatch.setattr("sparseflow_b200.nn.sparseflow_moe.SparseFlowMoE", lambda *args: made.append(args[5]))
    for block, want in ((_block(), True), (_block(norm_topk_prob=False), False), (_block(norm_topk_prob=True), True),
                        (_block(config=SimpleNamespace(norm_topk_prob=False)), False),
                        (_block(norm_topk_prob=True, config=SimpleNamespace(norm_topk_prob=False)), True)):
        make_sparseflow_moe(block)
        assert made.pop() is want
    for name in ("renormalize", "normalize_weights"):      # a name that is not known is not guessed at
        _refused(_block(**{name: False}), name)
        make_sparseflow_moe(_block(**{name: False}), renormalize=False)
        assert made.pop() is False
