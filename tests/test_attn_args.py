"""CPU: what the attention entry points refuse before they touch a GPU."""
import ctypes

import pytest
import torch


def config(pkg, **kw):
    c = dict(n_q_heads=16, n_kv_heads=2, head_dim=256, page_tokens=16, type=pkg.T_F16, max_seqs=8)
    c.update(kw)
    return pkg._AttnConfig(**c)


@pytest.mark.parametrize("kw, status", [
    (dict(head_dim=96), "MOE_EUNSUPPORTED"), (dict(head_dim=0), "MOE_EUNSUPPORTED"), (dict(type=0), "MOE_EUNSUPPORTED"),
    (dict(type=2), "MOE_EUNSUPPORTED"), (dict(n_q_heads=0), "MOE_EINVAL"), (dict(n_q_heads=257), "MOE_EINVAL"),
    (dict(n_q_heads=15), "MOE_EINVAL"), (dict(n_kv_heads=0), "MOE_EINVAL"), (dict(n_kv_heads=-2), "MOE_EINVAL"),
    (dict(n_kv_heads=32), "MOE_EINVAL"), (dict(page_tokens=8), "MOE_EINVAL"), (dict(page_tokens=24), "MOE_EINVAL"),
    (dict(page_tokens=2048), "MOE_EINVAL"), (dict(max_seqs=0), "MOE_EINVAL"), (dict(max_seqs=65536), "MOE_EINVAL")])
def test_create_refuses(pkg, kw, status):
    h = ctypes.c_void_p()
    cfg = config(pkg, **kw)
    assert pkg.lib().moe_attn_create(0, ctypes.byref(cfg), ctypes.byref(h)) == getattr(pkg, status)
    assert not h.value and pkg.lib().moe_last_error()


def test_null_arguments(pkg):
    L = pkg.lib()
    h = ctypes.c_void_p()
    cfg = config(pkg)
    assert L.moe_attn_create(0, None, ctypes.byref(h)) == pkg.MOE_EINVAL
    assert L.moe_attn_create(0, ctypes.byref(cfg), None) == pkg.MOE_EINVAL
    assert L.moe_attn_destroy(None) == pkg.MOE_EINVAL
    assert L.moe_kv_append(None, None, None, None, None, 1, 0, 0, None) == pkg.MOE_EINVAL
    assert L.moe_attn_decode(None, None, None, None, 0, 1.0, None, 0, None, None) == pkg.MOE_EINVAL
    assert L.moe_attn_prompt(None, None, None, None, 0, 1.0, None, 0, None, None) == pkg.MOE_EINVAL
    assert L.moe_attn_flags(None, None, None) == pkg.MOE_EINVAL
    assert L.moe_attn_flags_async(None, None, None) == pkg.MOE_EINVAL
    assert b"null" in L.moe_last_error()


def test_cache_and_batch_refuse(pkg):
    k = torch.zeros((3, 2, 16, 64), dtype=torch.float16)
    pkg.KVCache(k, k.clone())
    for a, b in [(k, k[:2]), (k, k.bfloat16()), (k.float(), k.float()), (k[0], k[0]),
                 (k, k.transpose(1, 2).contiguous().transpose(1, 2)), (k.transpose(2, 3), k.transpose(2, 3))]:
        with pytest.raises(ValueError):
            pkg.KVCache(a, b)
    pages, n = torch.zeros((2, 4), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    start = torch.zeros(3, dtype=torch.int32)
    assert pkg.SeqBatch(pages, n).n_rows == 2
    pkg.SeqBatch(pages, n, start, n_rows=0)
    for args, kw in [((pages.long(), n), {}), ((pages, n.long()), {}), ((pages, n[:1]), {}), ((pages[0], n), {}),
                     ((pages, n, start), {}), ((pages, n, start[:2]), dict(n_rows=2)), ((pages, n), dict(n_rows=3)),
                     ((pages.t(), torch.zeros(4, dtype=torch.int32)), {}),
                     ((pages, n, torch.zeros(6, dtype=torch.int32)[::2]), dict(n_rows=2))]:
        with pytest.raises(ValueError):
            pkg.SeqBatch(*args, **kw)


def test_context_refuses_dtype(pkg):
    with pytest.raises(ValueError):
        pkg.AttnContext(16, 2, 256, 16, 4, dtype=torch.float32)
