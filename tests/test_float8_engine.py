"""Serving in 8 bits, the parts that need no GPU: what the configuration and the engine refuse, and what a cache in 8 bits takes."""
import pytest
import torch

from garuda_b200.config.engine_config import EngineConfig
from garuda_b200.config.model_config import ConfigError
from tests.helpers import TINY, model_dir
from tests.plain.cpu_ops import CpuOps


def test_configuration():
    cfg = EngineConfig.from_dict({"model": {"weight_dtype": "float8_e4m3"}, "memory": {"cache_dtype": "float8_e4m3"}})
    assert cfg.model.weight_dtype == cfg.memory.cache_dtype == "float8_e4m3"
    assert EngineConfig.from_dict({}).memory.cache_dtype == ""
    for bad in ({"model": {"weight_dtype": "int8"}}, {"memory": {"cache_dtype": "float8"}},
                {"model": {"weight_dtype": "float8_e4m3", "dtype": "float32"}}, {"memory": {"cache_dtype": 8}}):
        with pytest.raises(ConfigError):
            EngineConfig.from_dict(bad)


def test_engine_refuses():
    from garuda_b200 import Engine
    for kw in (dict(weight_dtype="int8"), dict(cache_dtype="float16"), dict(weight_dtype="float8_e4m3", dtype="float32"),
               dict(weight_dtype="float8_e4m3"), dict(cache_dtype="float8_e4m3")):      # the last two: the plain kernel set knows neither
        with pytest.raises(ConfigError):
            Engine(model_dir("A"), **{"dtype": "bfloat16", "ops": CpuOps(), **kw})


def test_models_whose_layers_do_not_know_8_bits_are_refused():
    from garuda_b200.config.registry import build_model
    from garuda_b200.engine.engine import Engine
    from tests.murilorn_cases import CASES

    class Half:
        _check_float8 = Engine._check_float8
    half = Half()
    _, half.model = build_model(TINY["A"][0])
    half._check_float8(True, True)
    config = next(iter(CASES.values()))
    config = config[0] if isinstance(config, tuple) else config
    _, half.model = build_model(config)
    half._check_float8(False, False)
    for weights, cache in ((True, False), (False, True)):
        with pytest.raises(ConfigError):
            half._check_float8(weights, cache)


def test_pages_in_8_bits():
    from garuda_b200.cache.manager import CacheConfig, PagedCache
    from garuda_b200.config.registry import build_model
    _, model = build_model(TINY["D"][0])
    plain = PagedCache(model, CacheConfig(page_size=32, num_pages=3), torch.bfloat16, "cpu")
    small = PagedCache(model, CacheConfig(page_size=32, num_pages=3), torch.bfloat16, "cpu", float8=True)
    for a, b, ks, vs in zip(plain.k_pools, small.k_pools, small.k_scales, small.v_scales):
        assert b.shape == a.shape and b.dtype == torch.float8_e4m3fn
        assert ks.shape == vs.shape == a.shape[:3] and ks.dtype == torch.float32
    assert plain.bytes_per_position() < 2 * small.bytes_per_position() < 1.05 * plain.bytes_per_position()
    tables = [torch.zeros(1, 1, dtype=torch.int32)] * len(model.cache_groups)
    for cache in small.layer_caches(tables):
        assert cache.k_scale.shape == cache.v_scale.shape == cache.k.shape[:2]
    assert all(c.k_scale is None for c in plain.layer_caches(tables))


@pytest.mark.parametrize("head_dim,taken", [(16, True), (80, True), (256, True), (8, False), (20, False), (100, False), (272, False)])
def test_head_sizes_that_no_8_bit_kernel_takes_are_refused_when_the_engine_is_made(head_dim, taken):
    from garuda_b200.config.registry import build_model
    from garuda_b200.engine.engine import Engine

    class Half:
        _check_float8 = Engine._check_float8
    half = Half()
    _, half.model = build_model(dict(TINY["A"][0], head_dim=head_dim))
    half._check_float8(True, False)              # the weights know no heads
    if taken:
        half._check_float8(False, True)
    else:
        with pytest.raises(ConfigError, match=f"heads of {head_dim} channels"):
            half._check_float8(False, True)
