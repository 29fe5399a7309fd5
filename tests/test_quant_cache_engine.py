"""The engine's side of the 8-bit cache that needs no GPU: what is planned, counted and refused."""
import pytest
import torch

from ginfer_b200.cache.storage import CacheStorage, GroupLayout, plan_groups
from ginfer_b200.config.engine_config import EngineConfig
from ginfer_b200.ops import quant_cache as qc
from ginfer_b200.parts.base import PagedKVSpec, StateSpec


def test_groups_and_bytes():
    specs = {0: PagedKVSpec(2, 64, kept="int8"), 1: PagedKVSpec(2, 64, 48, kept="int8"),
             2: PagedKVSpec(2, 64, kept="int8"), 3: StateSpec((3,))}
    groups, where = plan_groups(specs)
    assert [g.cache_ids for g in groups] == [(0, 2), (1,)] and where == {0: 0, 2: 0, 1: 1}
    assert all(g.kept == "int8" for g in groups)
    # two caches, keys and values of 2 heads: 64 bytes of codes and 4 of scale a row
    assert groups[0].bytes_per_page(16, 2) == 2 * 16 * 2 * 2 * 68
    assert GroupLayout(((2, 64),) * 2, True, 0, (0, 2)).bytes_per_page(16, 2) == 2 * 16 * 2 * 2 * 128
    wide = [GroupLayout(((4, 128),) * 2, True, 0, (0,), 0, k).bytes_per_page(16, 2) for k in ("", "fp8")]
    assert wide[0] / wide[1] > 1.93                             # nearly twice the tokens of a bfloat16 cache


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_storage(kind):
    specs = {5: PagedKVSpec(3, 32, kept=kind), 7: PagedKVSpec(3, 32, kept=kind)}
    groups, _ = plan_groups(specs)
    st = CacheStorage(specs, groups, [9], 4, 2, torch.bfloat16, "cpu")
    for c in (5, 7):
        codes, scales = st.pages_of(c)
        facts = qc._cache((codes, scales))                      # a page more than the manager hands out
        assert facts[3:] == (10, 3, 4, 32) and codes.dtype == qc.KINDS[kind]
    assert st.pages_of(5)[0].data_ptr() != st.pages_of(7)[0].data_ptr()


def test_models_that_keep_other_things_are_refused():
    import ginfer_b200.architectures  # noqa: F401
    from ginfer_b200.config.registry import resolve_architecture
    from ginfer_b200.parts.model import DecoderModel
    from tiny import CONFIGS
    from tiny_bapivik import MIXED

    def model(config):
        arch = resolve_architecture(config)
        return DecoderModel(arch.build_plan(arch.config_cls.from_dict(config)))
    specs = model(CONFIGS["E"]).cache_specs_in_8_bits("fp8")
    assert [s.kept for s in specs.values()] == ["fp8"] * 2 and specs[1].window == 70
    with pytest.raises(ValueError, match="does not read a cache of 8 bits"):
        model(MIXED).cache_specs_in_8_bits("int8")
    odd = dict(CONFIGS["A"], head_dim=24)
    with pytest.raises(ValueError, match="multiple of 16"):
        model(odd).cache_specs_in_8_bits("int8")


def test_options():
    EngineConfig("x", kv_cache_dtype="fp8").validate()
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        EngineConfig("x", kv_cache_dtype="int4").validate()
    from ginfer_b200.cli import build_parser
    assert build_parser().parse_args(["--kv-cache-dtype", "int8"]).kv_cache_dtype == "int8"
    assert build_parser().parse_args([]).kv_cache_dtype == "auto"


@pytest.mark.parametrize("pages,page,want", [
    ([], 16, []), ([1], 16, [(0, 1)]), ([64] * 32, 16, [(0, 32)]), ([64] * 33, 16, [(0, 32), (32, 33)]),
    ([5000, 1, 1], 16, [(0, 1), (1, 3)]), ([1, 5000, 1], 16, [(0, 1), (1, 2), (2, 3)]),
    ([1024, 1024, 1025], 16, [(0, 2), (2, 3)]), ([2, 4, 8], 4096, [(0, 2), (2, 3)])])
def test_portions_are_read_back_in_groups(pages, page, want):
    assert qc.portion_groups(pages, page) == want
