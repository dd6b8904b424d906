"""The 4-bit cache's format: the oracle's codes by definition, the entry points' refusals on the host (CPU only)."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from oracle import paged_cache as oracle
from tests.conftest import import_package


def test_codes_are_the_nearest_and_ties_go_to_the_even_one():
    x = torch.zeros(32, dtype=torch.float64)
    x[:16] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 0.2500001, 0.7499999, -1.25, -2.5, -6.1, 6.9, 0.1, -0.1])
    codes, scales = oracle.encode(x)
    assert scales.tolist() == [127]
    want = [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, 0.5, 0.5, -1.0, -2.0, -6.0, 6.0, 0.0, 0.0]
    assert oracle.decode(codes, scales)[:16].tolist() == want


@pytest.mark.parametrize("top,e", [(7.0, 0), (math.nextafter(7.0, 8.0), 1), (0.0, -125), (2.0 ** -140, -125), (1.0, -2), (0.875, -3),
                                   (3.4028234663852886e38, 125), (7 * 2.0 ** 125, 125)])
def test_the_scale_is_the_smallest_that_holds(top, e):
    assert oracle.scale_exponents(torch.tensor([top], dtype=torch.float64)).tolist() == [e]


def test_no_value_is_off_by_more_than_the_scale():
    x = torch.randn(64, 64, generator=torch.Generator().manual_seed(0), dtype=torch.float64) * 3
    codes, scales = oracle.encode(x)
    off = (oracle.decode(codes, scales) - x).abs()
    assert (off <= 2.0 ** (scales.double() - 127).repeat_interleave(32, -1)).all()


def test_a_block_that_is_not_finite_reads_as_nan():
    x = torch.ones(2, 64)
    x[0, 3], x[1, 40] = math.inf, math.nan
    y = oracle.decode(*oracle.encode(x))
    assert torch.isnan(y).tolist() == [[True] * 32 + [False] * 32, [False] * 32 + [True] * 32]


def struct(lib_mod, **over):
    values = dict(data=16, log_mass=None, page_table=16, pages=4, page_size=64, kv_heads=2, head_dim=64, batch=1, table_width=2)
    return lib_mod.PagedCacheStruct(**{**values, **over})


BAD_CACHES = [dict(head_dim=32), dict(head_dim=96), dict(page_size=16), dict(page_size=48), dict(page_size=2048),
              dict(pages=-1), dict(kv_heads=0), dict(batch=-1), dict(table_width=-1), dict(table_width=1 << 30),
              dict(data=None), dict(data=8), dict(page_table=None)]


@pytest.mark.parametrize("over", BAD_CACHES)
def test_bad_caches_are_refused(over):
    lib_mod = import_package("_lib")
    lib = lib_mod.load()
    cache, size = struct(lib_mod, **over), ctypes.c_size_t()
    assert lib.vgo_cached_attn_workspace(ctypes.byref(cache), 2, 1, 0, 0, 1, ctypes.byref(size)) == lib_mod.VGO_EINVAL
    assert lib.vgo_cache_append(ctypes.byref(cache), ctypes.byref(lib_mod.CacheTokens()), 1, None) == lib_mod.VGO_EINVAL
    assert lib.vgo_cache_read(ctypes.byref(cache), 16, None, 1, 16, 16, 1, None) == lib_mod.VGO_EINVAL


def tokens(lib_mod, **over):
    strides = (ctypes.c_int64 * 3)(64, 64, 64)
    values = dict(k=16, v=16, q=None, q_out=None, heads=0, n_tokens=1, k_stride=strides, v_stride=strides, starts=16)
    return lib_mod.CacheTokens(**{**values, **over})


@pytest.mark.parametrize("over", [
    dict(n_tokens=-1), dict(n_tokens=1 << 31), dict(heads=-1), dict(heads=1 << 16), dict(starts=None), dict(k=None), dict(v=8),
    dict(heads=2), dict(heads=2, q=16), dict(rope_sin=16), dict(rope_cos=16), dict(positions=16), dict(log_mass=16),
    dict(rope_sin=4, rope_cos=16), dict(rope_sin=16, rope_cos=16, rope_rows=-1), dict(k_stride=(ctypes.c_int64 * 3)(64, 64, 3)),
    dict(v_stride=(ctypes.c_int64 * 3)(-64, 64, 64))])
def test_bad_tokens_are_refused(over):
    lib_mod = import_package("_lib")
    cache, bad = struct(lib_mod), tokens(lib_mod, **over)
    assert lib_mod.load().vgo_cache_append(ctypes.byref(cache), ctypes.byref(bad), 1, None) == lib_mod.VGO_EINVAL


def test_more_tokens_than_a_grid_has_threads_for():
    lib_mod = import_package("_lib")
    lib = lib_mod.load()
    cache, many = struct(lib_mod, batch=1 << 20, kv_heads=64), tokens(lib_mod, n_tokens=1 << 20)
    assert lib.vgo_cache_append(ctypes.byref(cache), ctypes.byref(many), 1, None) == lib_mod.VGO_EINVAL
    assert lib.vgo_cache_read(ctypes.byref(cache), 16, None, 1 << 20, 16, 16, 1, None) == lib_mod.VGO_EINVAL
    strides = (ctypes.c_int64 * 3)(64, 64, 64)
    assert lib.vgo_cached_attn_fwd(ctypes.byref(cache), 16, strides, 64, 1 << 20, 16, None, 0, 1.0, 16, strides, 1, None, 0,
                                   None) == lib_mod.VGO_EINVAL


@pytest.mark.parametrize("over", [dict(heads=3), dict(heads=0), dict(n_query=-1), dict(dtype=7), dict(scale=0.0), dict(scale=math.inf),
                                  dict(scale=math.nan), dict(q=None), dict(q=8), dict(out=None), dict(lengths=None)])
def test_bad_queries_are_refused(over):
    lib_mod = import_package("_lib")
    strides = (ctypes.c_int64 * 3)(64, 64, 64)
    v = {**dict(heads=2, n_query=1, dtype=1, scale=1.0, q=16, out=16, lengths=16), **over}
    cache = struct(lib_mod)
    status = lib_mod.load().vgo_cached_attn_fwd(
        ctypes.byref(cache), v["q"], strides, v["heads"], v["n_query"], v["lengths"], None, 0, v["scale"], v["out"], strides,
        v["dtype"], None, 0, None)
    assert status == lib_mod.VGO_EINVAL


def test_empty_calls_launch_nothing():
    lib_mod = import_package("_lib")
    lib = lib_mod.load()
    for over in (dict(batch=0),):
        cache = struct(lib_mod, **over)
        assert lib.vgo_cache_append(ctypes.byref(cache), ctypes.byref(tokens(lib_mod)), 1, None) == lib_mod.VGO_OK
        assert lib.vgo_cache_read(ctypes.byref(cache), None, None, 4, None, None, 1, None) == lib_mod.VGO_OK
    cache = struct(lib_mod)
    assert lib.vgo_cache_append(ctypes.byref(cache), ctypes.byref(tokens(lib_mod, n_tokens=0, k=None, v=None)), 1, None) == lib_mod.VGO_OK


def test_host_tensors_and_shapes_are_refused():
    vgo = import_package()
    cache = vgo.PagedCache.empty(4, 2, 64, device="cpu")
    assert cache.data.shape == (4, 2, 2, 34 * 64) and (cache.page_size, cache.kv_heads, cache.head_dim) == (64, 2, 64)
    assert vgo.PagedCache.empty(4, 2, 128, page_size=32, masses=True, device="cpu").log_mass.shape == (4, 32)
    table, one = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x = torch.zeros(1, 2, 1, 64)
    for call in (lambda: vgo.cache_append(cache, x, x, table, one), lambda: vgo.cache_read(cache, table, one, 1),
                 lambda: vgo.cached_attention(x, cache, table, one)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    for over in (dict(head_dim=96), dict(page_size=48), dict(page_size=16), dict(page_size=2048), dict(kv_heads=0), dict(pages=-1)):
        arguments = {**dict(pages=1, kv_heads=1, head_dim=64, device="cpu"), **over}
        with pytest.raises(ValueError):
            vgo.PagedCache.empty(**arguments)


@pytest.mark.parametrize("at", [17, 18])
def test_masses_that_are_no_floats_are_refused(at):
    """(Any float's address will do: the kernels' wide loads of masses ask for no more.)"""
    lib_mod = import_package("_lib")
    lib, size = lib_mod.load(), ctypes.c_size_t()
    status = lambda cache: lib.vgo_cached_attn_workspace(ctypes.byref(cache), 2, 1, 0, 0, 1, ctypes.byref(size))
    assert status(struct(lib_mod, log_mass=at)) == lib_mod.VGO_EINVAL
    assert status(struct(lib_mod, log_mass=20)) == lib_mod.VGO_OK


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_bounds_tell_two_terms_of_a_probability_from_one(dtype):
    """The two keys of the GPU's test of few queries: one bf16 number a probability is past the bound of two, two are not."""
    pages = oracle.Pages(1, 1, 64, 64)
    pages.k[0, 0, 0, 0], pages.v[0, 0, 0], pages.v[0, 0, 1] = 1.0, 1.0, -2.0
    q = torch.zeros(1, 1, 40, 64)
    q[..., 0] = 0.6796875 + torch.arange(40) * 2.0 ** -8
    q = q.to(dtype)
    table, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.tensor([2], dtype=torch.int32)
    want, bound = oracle.attention(q, pages, table, lengths, scale=1.0, p_bits=2.0 ** -16)
    p = torch.stack([torch.ones(40, dtype=torch.float64), torch.exp(-q[0, 0, :, 0].double())])
    one = p.bfloat16().double()
    two = one + (p - one).bfloat16().double()
    off = lambda t: ((t[0] - 2 * t[1]) / p.sum(0) - want[0, 0, :, 0]).abs() - bound[0, 0, :, 0]
    assert off(two).max() <= 0 and off(one)[0] > 0 and (off(one) > 0).sum() > 30  # (some are bf16 numbers, nearly)


@pytest.mark.parametrize("over", [dict(n_query=1 << 30, heads=64), dict(batch=1 << 30, n_query=1 << 30, heads=65534, kv_heads=32767),
                                  dict(batch=(1 << 31) - 1, n_query=(1 << 31) - 1, heads=65535, kv_heads=65535)])
def test_a_workspace_is_asked_for_what_can_be_run(over):
    """The sizes that the attention itself refuses are refused here, too, before they overflow 64 bits."""
    lib_mod = import_package("_lib")
    v = {**dict(batch=1, kv_heads=2, heads=2, n_query=1), **over}
    cache, size = struct(lib_mod, batch=v["batch"], kv_heads=v["kv_heads"]), ctypes.c_size_t(7)
    status = lib_mod.load().vgo_cached_attn_workspace(ctypes.byref(cache), v["heads"], v["n_query"], 0, 0, 1, ctypes.byref(size))
    assert status == lib_mod.VGO_EINVAL
