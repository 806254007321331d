"""A sequence cache in 8 bits, what the host decides: which models and rows have it, what a fork copies, what it takes in memory."""
import pytest
import torch

from qwenforge_b200 import ops
from qwenforge_b200.cache import PAGE_TOKENS, KvNeed, SequenceCache
from qwenforge_b200.config import config_from_dict, preset_config, resolve_cache_dtype
from qwenforge_b200.engine import Model
from qwenforge_b200.ops import KernelError
from tests import helpers

CODES = torch.float8_e4m3fn


def test_names():
    assert resolve_cache_dtype(None) is None and resolve_cache_dtype("auto") is None
    assert resolve_cache_dtype("float8_e4m3") is CODES and resolve_cache_dtype(CODES) is CODES
    for wrong in ("int8", "bfloat16", torch.bfloat16, torch.float8_e5m2):
        with pytest.raises(ValueError):
            resolve_cache_dtype(wrong)


@pytest.mark.parametrize("name", ["mefepel-tiny", "zebovik-tiny", "rarevik-tiny", "gatosun-tiny", "dapupel-tiny", "lasonex-tiny", "tiny-b"])
def test_models_whose_attention_has_no_such_form(name):
    """(tiny-b: heads of 24)"""
    with pytest.raises(ValueError, match="float8_e4m3"):
        Model(preset_config(name).model_spec(), torch.float32, "cpu", cache_dtype="float8_e4m3")


@pytest.mark.parametrize("name", ["qwen2.5-0.5b", "qwen2.5-3b", "qwen2.5-7b", "tiny-a"])
def test_models_that_have_it(name):
    assert Model(preset_config(name).model_spec(), torch.float32, "cpu", cache_dtype="float8_e4m3").cache_dtype is CODES
    assert Model(config_from_dict(helpers.TINY_W).model_spec(), torch.float32, "cpu", cache_dtype=CODES).cache_dtype is CODES


def test_rows_that_fit():
    assert KvNeed(2, 64).fits(CODES) and KvNeed(2, 16, window=37).fits(CODES)
    for need in (KvNeed(2, 24), KvNeed(2, 256), KvNeed(2, 64, planes=1), KvNeed(2, 64, chunk=8), KvNeed(2, 64, every=4), KvNeed(2, 64, window=8, pool=4)):
        assert not need.fits(CODES)
        with pytest.raises(ValueError):
            SequenceCache([need], 4 * PAGE_TOKENS, 2, 4 * PAGE_TOKENS, torch.float32, "cpu", CODES)
    assert not KvNeed(2, 64).fits(torch.bfloat16)


def test_memory():
    needs = [KvNeed(2, 64), KvNeed(2, 64), KvNeed(3, 32, window=70)]
    cache = SequenceCache(needs, 10 * PAGE_TOKENS, 4, 6 * PAGE_TOKENS, torch.bfloat16, "cpu", CODES)
    a, b = cache.kv_groups
    assert a.storage.dtype is CODES and a.storage.shape == (2, 10, 2, 2, 64, 64) and a.scales.shape == (2, 10, 2, 2)
    assert a.values.dtype is torch.bfloat16 and a.values.shape == (10, 2, 2, 64, 64) and not bool(a.values.any())
    # codes, scales, and one entry's values beside them
    assert cache.storage_bytes() == sum(g.storage.numel() + 4 * g.scales.numel() + 2 * g.values.numel() for g in (a, b))
    assert cache.read_bytes([100]) == 2 * 100 * 2 * 2 * 64 + 70 * 2 * 3 * 32
    assert cache.site(1).scales.data_ptr() == a.scales[1].data_ptr() and cache.site(2).scales.shape == (10, 2, 3)
    plain = SequenceCache(needs, 10 * PAGE_TOKENS, 4, 6 * PAGE_TOKENS, torch.bfloat16, "cpu")
    assert plain.kv_dtype is None and plain.site(0).scales is None and plain.kv_groups[0].values is None
    assert plain.read_bytes([100]) == 2 * cache.read_bytes([100])


def test_scales_travel_with_their_pages(monkeypatch):
    copies = []
    monkeypatch.setattr(ops, "copy_pages", lambda storage, moves: copies.append((storage, list(moves))))
    cache = SequenceCache([KvNeed(2, 64)], 20 * PAGE_TOKENS, 6, 8 * PAGE_TOKENS, torch.float32, "cpu", CODES)
    group = cache.kv_groups[0]
    first, slot = cache.open(), cache.open()
    for s, n in ((first, 200), (slot, 100)):
        cache.reserve([(s, n)])
        cache.advance(s, n)
    forks = cache.fork(slot, 2)
    (a, rows), (b, whole) = copies
    assert a is group.storage and b is group.scales and [m[2] for m in rows] == [36, 36] and whole == [m[:2] for m in rows]
    copies.clear()
    cache.rewind(forks[0], 50)    # into the page that the three of them share
    assert [c[0] is group.scales for c in copies] == [False, True] and copies[1][1] == [copies[0][1][0][:2]]
    copies.clear()
    cache.close(first)
    assert cache.compact() > 0
    assert len(copies) == 2 and copies[0][1] == copies[1][1] and copies[1][0] is group.scales
    assert cache.shared_worth_reading([slot, *forks]) is None


def test_what_is_on_the_cpu_is_refused():
    storage, table = torch.zeros((2, 2, 1, 64, 64), dtype=torch.uint8).view(CODES), torch.zeros((1, 2), dtype=torch.int32)
    with pytest.raises(KernelError, match="CUDA"):
        ops.E4m3SiteArgs(storage, torch.zeros((2, 2, 1)), table, 1, 64)


def test_which_steps_attend_over_codes():
    assert ops.attention_e4m3_pays(torch.bfloat16, 1, 7) and ops.attention_e4m3_pays(torch.bfloat16, 16, 8)
    assert not ops.attention_e4m3_pays(torch.bfloat16, 17, 8) and ops.attention_e4m3_pays(torch.float32, 2048, 7)
