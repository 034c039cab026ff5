"""Serving a model in few bits: its keys and values in 8, its layers' matrices in 4.

`in_few_bits` turns a model's description into that of the same model so served; which parts can be is said here, by kind.
Embedding, output head and norms stay as they are.
"""
from __future__ import annotations

import dataclasses
from typing import Optional

from .schema import ConfigError, ModelSpec, PartSpec

CACHE_KINDS = ("attention",)                   # mixers whose keys and values may be held in 8 bits
WEIGHT_KINDS = ("attention", "swiglu")         # parts whose matrices may be held in 4 bits
WEIGHT_GROUPS = (32, 64, 128)


def _with(part: PartSpec, **params) -> PartSpec:
    return PartSpec.make(part.kind, **{**part.as_dict(), **params})


def serves_few_bits(spec: ModelSpec) -> bool:
    """Whether any of a description's layers holds its keys and values in 8 bits or matrices in 4."""
    parts = [part for layer in spec.layers for part in (layer.mixer, layer.feed_forward) if part is not None]
    return any((part.kind in CACHE_KINDS and part.get("cache") is not None) or (part.kind in WEIGHT_KINDS and part.get("weights") is not None) for part in parts)


def in_few_bits(spec: ModelSpec, *, cache: Optional[str] = None, weights: Optional[str] = None, weight_group: int = 128) -> ModelSpec:
    """`cache` "e4m3": keys and values in float8 e4m3 with a power of two per block of 16 tokens and head (ops.PagedE4M3).
    `weights` "int4": the layers' matrices rounded to 4 bits with a scale per `weight_group` neighbouring inputs
    (ops.Int4Weight). None leaves them in the serving type."""
    if cache is None and weights is None:
        return spec
    if cache not in (None, "e4m3"):
        raise ConfigError(f"the cache is held in the serving type (None) or in 'e4m3', not {cache!r}")
    if weights not in (None, "int4"):
        raise ConfigError(f"weights are held in the serving type (None) or in 'int4', not {weights!r}")
    if weights is not None and weight_group not in WEIGHT_GROUPS:
        raise ConfigError(f"weights in 4 bits have a scale for each group of {WEIGHT_GROUPS}, not {weight_group!r}")
    layers = []
    for number, layer in enumerate(spec.layers):
        mixer, feed_forward = layer.mixer, layer.feed_forward
        if cache is not None:
            if mixer.kind not in CACHE_KINDS:
                raise ConfigError(f"layer {number}: the cache of a '{mixer.kind}' mixer cannot be held in 8 bits (only that of {CACHE_KINDS})")
            mixer = _with(mixer, cache=cache)
        if weights is not None:
            for part in (mixer, feed_forward):
                if part is not None and (part.kind not in WEIGHT_KINDS or part.get("bias")):
                    raise ConfigError(f"layer {number}: the matrices of '{part.kind}' cannot be held in 4 bits (only those of {WEIGHT_KINDS}, without "
                                      "biases in the feed-forward)")
            mixer = _with(mixer, weights=weights, weight_group=weight_group)
            feed_forward = None if feed_forward is None else _with(feed_forward, weights=weights, weight_group=weight_group)
        layers.append(dataclasses.replace(layer, mixer=mixer, feed_forward=feed_forward))
    return dataclasses.replace(spec, layers=tuple(layers))
