"""More refusals of the int4 cache's attention, without a GPU: arguments near the ends of their ranges."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from jacq_amd import kivi  # noqa: E402
from tests.test_kivi_attend import (CU, EINVAL, ENOMEM, GOOD, LENS, TABLES, attend,  # noqa: E402
                                    cpu_cache, error, q)


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_a_scale_that_is_infinite_in_base_two_is_refused(scale):
    """Scores are taken to base two, by scale x log2(e) in fp32."""
    error(attend(scale=scale), EINVAL, "finite")


@pytest.mark.parametrize("call", ["prefill", "cross"])
def test_a_scale_beyond_fp32_is_refused(call):
    with pytest.raises(kivi.KiviCheckError, match="SCALE"):
        getattr(cpu_cache(), call)(q(), CU, 2, LENS, TABLES, scale=1e39)


@pytest.mark.parametrize("call", ["prefill", "cross"])
def test_the_queries_of_one_head_may_lie_apart(call):
    """Heads of which there is one lie side by side whatever their stride is."""
    geo = kivi.KiviGeometry(1, 1, 64, 16, 32, 64, 8, 16)
    cache = kivi.PagedKiviCache(geo, 2, device="cpu")
    wide = torch.zeros((3, 96), dtype=torch.float16)
    for x in (wide[:, None, :64], wide[:, :64].unflatten(1, (1, 64)), wide[None, :, :64].transpose(0, 1)):
        assert x.shape == (3, 1, 64) and not x.is_contiguous()
        with pytest.raises(kivi.KiviCheckError, match="GPU device"):  # and nothing else is wrong
            getattr(cache, call)(x, CU, 2, LENS, TABLES)


@pytest.mark.parametrize("heads", [(40, 8, 128), (16, 16, 128), (64, 4, 64)])
@pytest.mark.parametrize("batch,tokens,chunk", [
    (2048, 32768, 8192), (1024, 131072, 16384), (2048, 131072, 32768), (65535, 8192, 2048),
    (65535, 262000, 8192), (30000, 131072, 20000)])
def test_a_chunk_beside_single_queries_is_taken_under_a_wide_table(heads, batch, tokens, chunk):
    """Whatever the table's width and max_q x sequences; no workspace is given, so nothing is launched."""
    geo = dict(num_heads=heads[0], num_kv_heads=heads[1], head_dim=heads[2], max_pages_per_seq=tokens // 16)
    total = batch - 1 + chunk
    size = kivi.lib().jacq_kivi_attend_workspace_size(kivi.KiviGeometry(**{**GOOD, **geo}).ref, batch, total,
                                                      chunk)
    assert 0 < size < 2 ** 33
    rc = attend(geo=geo, batch=batch, total_q=total, max_q=chunk, q_stride=heads[0] * heads[2])
    error(rc, ENOMEM, str(size))


def test_many_long_chunks_are_taken_under_a_wide_table():
    """More blocks of 32 rows than a launch has workgroups, but not more row tiles; nothing is launched."""
    geo = dict(num_heads=16, num_kv_heads=1, head_dim=64, max_pages_per_seq=16384 // 16)
    kw = dict(batch=65535, total_q=65535 * 520, max_q=520)
    size = kivi.lib().jacq_kivi_attend_workspace_size(kivi.KiviGeometry(**{**GOOD, **geo}).ref, *kw.values())
    assert 0 < size < 2 ** 33
    error(attend(geo=geo, q_stride=16 * 64, **kw), ENOMEM, str(size))
