"""Serving in few bits as a matter of a model's description, on the CPU."""
import pytest
import torch

from tiny_configs import TINY_A
from vosti_b200 import Engine
from vosti_b200.cache import CacheManager
from vosti_b200.config import ConfigError, PartSpec, in_few_bits, model_spec_from_config, serves_few_bits
from vosti_b200.models import build_model
from vosti_b200.parts import build_feed_forward, build_mixer


def test_what_a_description_becomes():
    spec = model_spec_from_config(TINY_A)
    assert in_few_bits(spec) is spec
    few = in_few_bits(spec, cache="e4m3", weights="int4", weight_group=64)
    for before, layer in zip(spec.layers, few.layers):
        assert layer.mixer.get("cache") == "e4m3" and layer.mixer.get("weights") == layer.feed_forward.get("weights") == "int4"
        assert layer.mixer.get("weight_group") == layer.feed_forward.get("weight_group") == 64
        assert before.mixer.get("cache") is None and layer.norm == before.norm and layer.position == before.position
    model = build_model(few)
    assert model.expected_weights().keys() == build_model(spec).expected_weights().keys()
    caches, _ = model.cache_specs()
    assert all(c.storage == "e4m3" for c in caches)
    only = in_few_bits(spec, cache="e4m3")
    assert only.layers[0].mixer.get("weights") is None and only.layers[0].feed_forward == spec.layers[0].feed_forward


@pytest.mark.parametrize("bad", [dict(cache="int8"), dict(cache="float8"), dict(weights="int8"), dict(weights="int4", weight_group=16), dict(weights="int4", weight_group=256)])
def test_unknown_forms(bad):
    with pytest.raises(ConfigError):
        in_few_bits(model_spec_from_config(TINY_A), **bad)


def test_models_whose_parts_cannot():
    from tiny_beralix import ALL
    for raw, _ in ALL.values():
        spec = model_spec_from_config(raw)
        for form in (dict(cache="e4m3"), dict(weights="int4")):
            with pytest.raises(ConfigError, match="cannot be held"):
                in_few_bits(spec, **form)


def test_parts_refuse():
    sizes = dict(num_heads=2, num_kv_heads=1, head_dim=64, scale=0.125)
    with pytest.raises(ConfigError):
        build_mixer(PartSpec.make("attention", cache="int8", **sizes), 128, None)
    with pytest.raises(ConfigError):
        build_mixer(PartSpec.make("attention", weights="int8", **sizes), 128, None)
    with pytest.raises(ConfigError):
        build_feed_forward(PartSpec.make("swiglu", intermediate_size=64, weights="int4", bias=True, activation="clamped", limit=7.0, sigmoid_scale=1.7), 128)
    part = build_feed_forward(PartSpec.make("swiglu", intermediate_size=64, weights="int4"), 128)
    tensors = {name: torch.zeros(w.shape) for name, w in part.weight_specs().items()}
    with pytest.raises(RuntimeError, match="bfloat16"):
        part.load(tensors, torch.float32)


def test_engine_refuses():
    for mode in (True, "full", "decode"):
        with pytest.raises(ValueError, match="batch_invariant"):
            Engine("nowhere", cache_dtype="e4m3", batch_invariant=mode)
        with pytest.raises(ValueError, match="batch_invariant"):
            Engine("nowhere", weights="int4", batch_invariant=mode)
    with pytest.raises(ValueError, match="bfloat16"):
        Engine("nowhere", weights="int4", dtype="float32")


@pytest.mark.parametrize("form", [dict(cache="e4m3"), dict(weights="int4"), dict(cache="e4m3", weights="int4")])
def test_engine_refuses_a_description_in_few_bits(form):
    """The same as by the engine's own arguments."""
    plain = model_spec_from_config(TINY_A)
    few = in_few_bits(plain, **form)
    assert serves_few_bits(few) and not serves_few_bits(plain)
    for mode in (True, "1", "full", "decode"):
        with pytest.raises(ValueError, match="batch_invariant"):
            Engine(spec=few, tensors={}, num_blocks=4, batch_invariant=mode)


def test_pages_hold_whole_blocks():
    caches, states = build_model(in_few_bits(model_spec_from_config(TINY_A), cache="e4m3")).cache_specs()
    with pytest.raises(ValueError, match="16"):
        CacheManager(caches, states, num_pages=4, page_size=8, max_requests=1)
    CacheManager(caches, states, num_pages=4, page_size=32, max_requests=1)
