"""Matrices in 4 bits and keys and values in 8 (no GPU): what is offered and refused, what the cache manager keeps for 8-bit pages,
and which tiles of them a step's portions see."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from air_b200.cache.manager import CacheManager
from air_b200.config import ConfigError
from air_b200.csrc import ops
from air_b200.engine.engine import Engine, EngineConfig
from air_b200.parts.attention import held_tiles, plan_portions
from air_b200.parts.base import PagedKV, PagedKV8, SlotState
from air_b200.weights.loader import LoadReport


@pytest.mark.parametrize("formats", [{"weights": "int4"}, {"cache": "e5m2"}, {"weights": "mxfp4", "dtype": torch.float32},
                                     {"cache": "e4m3", "dtype": torch.float32}, {"weights": "mxfp4", "activation_terms": 0},
                                     {"weights": "mxfp4", "activation_terms": 4}])
def test_formats_that_are_refused(formats):
    with pytest.raises(ConfigError):
        EngineConfig(**formats).check_formats()


@pytest.mark.parametrize("formats", [{}, {"weights": "mxfp4"}, {"weights": "mxfp4", "activation_terms": 3, "cache": "e4m3"}, {"cache": "e4m3"}])
def test_formats_that_are_taken(formats):
    EngineConfig(**formats).check_formats()


@pytest.mark.parametrize("needs,formats", [([(PagedKV(2, 64),)], {"cache": "e4m3"}), ([(SlotState((4,)),)], {"cache": "e4m3"}),
                                           ([(PagedKV8(2, 64), PagedKV8(2, 64).scales), (PagedKV(2, 64),)], {"cache": "e4m3"}),
                                           ([(PagedKV(2, 64),)], {"weights": "mxfp4"})])
def test_models_that_have_no_such_form(needs, formats):
    model = SimpleNamespace(rt=SimpleNamespace(in_four_bits={}), cache_needs=lambda: needs)
    with pytest.raises(ConfigError, match="no matrix|8-bit form|no layer"):
        Engine(model, EngineConfig(**formats))


def test_pages_and_their_scales_are_one_group():
    pages, win = PagedKV8(2, 64), PagedKV8(2, 64, 40)
    needs = [(pages, pages.scales), (win, win.scales), (pages, pages.scales)]
    m = CacheManager(needs, 32, 6, 2, dtype=torch.bfloat16, max_blocks=8)
    assert [g.runs for g in m.groups] == [[0, 2], [1]]
    kv, scales = m.views(0)
    assert kv.kv.shape == (6, 2, 2, 32, 64) and kv.kv.dtype == torch.float8_e4m3fn
    assert scales.scales.shape == (6, 2, 2, 2) and scales.scales.dtype == torch.float32 and kv.group == scales.group == 0
    assert m.views(1)[1].group == 1 and m.views(2)[0].kv.data_ptr() != kv.kv.data_ptr()
    per_page = 2 * 2 * 32 * 64 + 2 * 2 * 2 * 4
    assert CacheManager.bytes_per_page(needs, 32, torch.bfloat16) == 3 * per_page
    m.open("a")
    m.reserve([("a", 120)])
    m.commit("a", 120)
    full, window = m.sequences["a"].pages
    assert all(p >= 0 for p in full) and [p >= 0 for p in window] == [False, False, True, True]      # keys below 81 are out of reach
    m.check()
    m.close("a")
    assert m.free_pages() == 6


@pytest.mark.parametrize("window", [None, 1, 64, 100])
def test_tiles_that_portions_see(window):
    counts, before, slots = [1, 64, 200, 3], [0, 100, 63, 640], [5, 0, 2, 9]
    held = held_tiles(counts, before, slots, window)
    assert held.dtype == np.int32
    want = []
    for n, b, slot in zip(counts, before, slots):
        lowest = min(max(0, p - window + 1) if window else 0 for p in range(b, b + n))
        seen = sorted({k // 64 for p in range(b, b + n) for k in range(max(0, p - window + 1) if window else 0, p + 1)})
        want += [(slot, t, lowest, b + n) for t in seen]
    assert [tuple(r) for r in held.tolist()] == want
    assert held_tiles([], [], [], window).shape == (0, 4)


def test_a_plan_of_portions():
    plan = plan_portions([300, 2], [0, 500], [1, 0], 4, None, "cpu")
    assert isinstance(plan.tiles, ops.PortionTiles)
    assert plan.tiles.tiles.dtype == torch.int32 and plan.tiles.tiles.shape[1] == 4 and plan.tiles.tiles.shape[0] % ops.TILE_PAIR == 0
    assert np.array_equal(plan.tiles.held.numpy(), held_tiles([300, 2], [0, 500], [1, 0], None))
    empty = plan_portions([], [], [], 4, None, "cpu")
    assert empty.tiles.tiles.shape == (0, 4) and empty.tiles.held.shape == (0, 4) and empty.segments is None


@pytest.mark.parametrize("n,k", [(128, 256), (4608, 3584), (37888, 3584), (640, 2048), (1, 32), (5120, 13824)])
def test_parts_of_a_product(n, k):
    parts, steps = ops.mxfp4_splits(n, k), -(-k // 256)
    per = -(-steps // parts)
    assert 1 <= parts <= steps and (parts - 1) * per < steps      # none without a step
    assert parts == 1 or per >= 2


def test_shapes_of_rows_in_four_bits():
    assert ops._mxfp4_shapes(130, 544, 2) == ((2, 130, 272), (2, 2, 6, 32, 16))
    for k, terms in ((0, 1), (48, 1), (64, 0), (64, 4)):
        with pytest.raises(ops.KernelError):
            ops._mxfp4_shapes(4, k, terms)


def test_what_a_report_says():
    r = LoadReport(in_four_bits={"a": 0.11, "b": 0.125})
    assert r.summary() == "2 matrices were rounded to microscaled 4-bit floating point, b the furthest: off by 12.5% of its root mean square"


@pytest.mark.parametrize("owns", [True, False])
def test_pages_of_another_run_are_read_behind_the_wait(owns, monkeypatch):
    """A step of single tokens asks for old keys and values ahead of the q/k/v product's end only where none of them was written in
    this step: not those of another run's layer."""
    from air_b200.parts.attention import Attention
    heads, kv_heads, d, T = 4, 2, 64, 3
    part = object.__new__(Attention)
    part.heads, part.kv_heads, part.head_dim, part.window, part.scale, part.bias, part.eight = heads, kv_heads, d, None, 0.125, None, True
    part.rt = SimpleNamespace(dtype=torch.bfloat16, page_tokens=64, is_fp32=False)
    part.position = SimpleNamespace(table=lambda: torch.zeros(8, d))
    width = (heads + 2 * kv_heads) * d
    product = lambda n: type("Product", (), {"small": lambda self, x: True, "partial": lambda self, x: torch.zeros(1, T, n),
                                             "__call__": lambda self, x, dtype: torch.zeros(T, n, dtype=dtype)})()
    part.qkv, part.q_only, part.o = product(width), product(heads * d), product(32)
    seen = []
    monkeypatch.setattr(ops, "empty", lambda shape, dtype, device: torch.empty(shape, dtype=dtype))
    monkeypatch.setattr(ops, "decode_attention8_fresh", lambda *a, **kw: seen.append((kw["write_kv"], kw["early"])))
    ctx = SimpleNamespace(all_decode=True, block_tables=[None], token_seq=None, positions=None, status=None)
    part.forward(torch.zeros(T, 32), ctx, (SimpleNamespace(kv=None, group=0), SimpleNamespace(scales=None)), owns_cache=owns)
    assert seen == [(owns, owns)]


@pytest.mark.parametrize("needs,copied", [([PagedKV8(4, 128)] * 2, 4 * 128), ([PagedKV8(2, 64, 100), PagedKV8(8, 128), PagedKV8(2, 64)], 8 * 128),
                                          ([PagedKV(4, 128)] * 2, 0)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_the_pool_leaves_room_for_what_a_step_copies(needs, copied, page, monkeypatch):
    """Every page seen by portions of one step, of as many requests as there may be, is copied to 16 bits, a layer at a time."""
    free, requests = 40 << 30, 24
    runs = [(n, n.scales) if isinstance(n, PagedKV8) else (n,) for n in needs]
    model = SimpleNamespace(rt=SimpleNamespace(device=None, dtype=torch.bfloat16), cache_needs=lambda: runs,
                            spec=SimpleNamespace(max_positions=1 << 30))
    monkeypatch.setattr(torch.cuda, "empty_cache", lambda: None)
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device: (free, free))
    pages = Engine._pages_that_fit(model, EngineConfig(page_tokens=page, max_requests=requests, max_tokens=None, memory_fraction=0.9))
    kept = CacheManager.bytes_per_page(runs, page, torch.bfloat16)
    # the worst case: requests of as many tokens as they hold, in tiles of 64, an unfinished one at either end
    copy = lambda n: (n * page // 64 + 2 * requests) * 64 * 2 * copied * 2
    assert pages * kept + copy(pages) <= 0.9 * free < (pages + 2) * kept + copy(pages + 2) + (1 << 20)


def test_no_room_for_a_page(monkeypatch):
    runs = [(PagedKV8(4, 128), PagedKV8(4, 128).scales)]
    model = SimpleNamespace(rt=SimpleNamespace(device=None, dtype=torch.bfloat16), cache_needs=lambda: runs,
                            spec=SimpleNamespace(max_positions=1024))
    monkeypatch.setattr(torch.cuda, "empty_cache", lambda: None)
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device: (1 << 20, 1 << 30))
    with pytest.raises(RuntimeError, match="a cache page takes"):
        Engine._pages_that_fit(model, EngineConfig(max_requests=4, max_tokens=None))


def test_portions_of_one_request_share_its_tiles():
    held = held_tiles([64, 37, 5, 0], [10, 74, 300, 7], [3, 3, 1, 2], 40).tolist()
    assert held == [[3, 0, 0, 111], [3, 1, 0, 111], [1, 4, 261, 305]]
    assert held_tiles([5, 64, 37], [300, 74, 10], [1, 3, 3], None).tolist() == [[1, t, 0, 305] for t in range(5)] + [[3, t, 0, 138] for t in range(3)]
