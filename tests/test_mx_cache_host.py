"""The MX cache's refusals, without a GPU: the Python entry points' checks of arguments and the C entry
points' (which return before they touch the HIP runtime; the pointers are never dereferenced)."""

import os

import numpy as np
import pytest
import torch

from tests import _mx_cache as R
from velograd_amd import _lib
from velograd_amd import kernels as vk


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from velograd_amd.build import build_library
        build_library()
    return _lib.load()


def _cache(fmt="e2m1", pages=3, page=16, kv=2, dim=64):
    return vk.mx_cache(pages, page, kv, dim, fmt, device="cpu")


def _i64(n):
    return torch.zeros(n, dtype=torch.int64)


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_an_empty_cache_has_the_documented_layout():
    c = vk.mx_cache(3, 32, 2, 128, "e2m1", device="cpu")
    assert c.k_codes.shape == (3, 2, 32, 64) and c.k_codes.dtype == torch.float4_e2m1fn_x2
    assert c.v_scales.shape == (3, 2, 4, 32) and c.v_scales.dtype == torch.float8_e8m0fnu
    c = vk.mx_cache(3, 32, 2, 128, "e4m3", device="cpu")
    assert c.v_codes.shape == (3, 2, 32, 128) and c.v_codes.dtype == torch.float8_e4m3fn
    parts = R.as_bytes(c)
    assert all((p == 0).all() for p in parts)
    assert (R.values(parts[0], np.swapaxes(parts[1], 2, 3), "e4m3") == 0).all()


@pytest.mark.parametrize("args", [
    (3, 16, 2, 64, "int4"), (3, 24, 2, 64, "e2m1"), (3, 8, 2, 64, "e2m1"), (3, 65536, 2, 64, "e2m1"),
    (3, 16, 2, 96, "e2m1"), (3, 16, 0, 64, "e2m1"), (-1, 16, 2, 64, "e2m1"),
])
def test_mx_cache_refuses(args):
    with pytest.raises(ValueError):
        vk.mx_cache(*args, device="cpu")


def test_rope_table_refuses():
    for args in ((-1, 64), (4, 63), (4, 0), (4, 64, 0.0), (4, 64, float("nan"))):
        with pytest.raises(ValueError):
            vk.rope_table(*args, device="cpu")


def test_cpu_tensors_are_refused():
    c, x = _cache(), torch.zeros(5, 2, 64)
    for call in (lambda: vk.mx_cache_write(x, x, c, _i64(5)),
                 lambda: vk.rope_mx_cache_write(x, x, x, torch.zeros(4, 64), _i64(5), c, _i64(5)),
                 lambda: vk.mx_cache_read(c, _i64(5)),
                 lambda: vk.mx_cache_attention(x, c, _i32(5, 2), _i32(5))):
        with pytest.raises(TypeError, match="ROCm"):
            call()


def _bad_caches():
    c = _cache()
    yield TypeError, list(c)
    yield TypeError, c[:3]
    yield TypeError, (None,) + c[1:]
    yield TypeError, (c.k_codes.view(torch.uint8),) + c[1:]
    yield TypeError, c[:1] + (c.k_scales.view(torch.uint8),) + c[2:]
    yield TypeError, c[:2] + (torch.zeros(3, 2, 16, 32).to(torch.float8_e4m3fn),) + c[3:]
    yield ValueError, c[:3] + (_cache(page=32).v_scales,)
    yield ValueError, c[:2] + (_cache(pages=4).v_codes,) + c[3:]
    yield ValueError, (c.k_codes[0],) + c[1:]
    yield ValueError, _cache(dim=128)[:1] + c[1:]
    yield ValueError, (torch.zeros(3, 2, 16, 48, dtype=torch.uint8).view(torch.float4_e2m1fn_x2),) + c[1:]
    yield ValueError, tuple(t.view(torch.uint8).transpose(0, 1).contiguous().transpose(0, 1).view(t.dtype) for t in c)
    yield ValueError, (c.k_codes.to("meta"),) + c[1:]


@pytest.mark.parametrize("at", range(13))
def test_bad_caches_are_refused(at):
    error, cache = list(_bad_caches())[at]
    x = torch.zeros(5, 2, 64)
    for call in (lambda: vk.mx_cache_write(x, x, cache, _i64(5)), lambda: vk.mx_cache_read(cache, _i64(5)),
                 lambda: vk.mx_cache_attention(x, cache, _i32(5, 2), _i32(5))):
        with pytest.raises(error):
            call()


X = torch.zeros(5, 2, 64)


@pytest.mark.parametrize("error,kw", [
    (TypeError, dict(k=X.double())), (TypeError, dict(v=X.half())), (TypeError, dict(k=X.numpy())),
    (ValueError, dict(k=X[:, :1])), (ValueError, dict(k=X[..., :32])), (ValueError, dict(v=X[:4])),
    (ValueError, dict(k=X[0])), (TypeError, dict(slots=_i32(5))), (ValueError, dict(slots=_i64(4))),
    (ValueError, dict(slots=_i64(5)[:, None])),
    (TypeError, dict(positions=_i32(5))), (ValueError, dict(positions=_i64(6))), (TypeError, dict(positions=None)),
    (TypeError, dict(cos_sin=torch.zeros(4, 64).double())), (ValueError, dict(cos_sin=torch.zeros(4, 32))),
    (TypeError, dict(cos_sin=None)), (TypeError, dict(q=X.half())), (ValueError, dict(q=X[:3])),
    (ValueError, dict(q=torch.zeros(5, 4, 128))),
])
def test_writes_refuse(error, kw):
    args = dict(q=X, k=X, v=X, cos_sin=torch.zeros(4, 64), positions=_i64(5), cache=_cache(), slots=_i64(5))
    args.update(kw)
    with pytest.raises(error, match="^(?!.*ROCm)"):
        vk.rope_mx_cache_write(**args)
    if not {"positions", "cos_sin", "q"} & set(kw):
        with pytest.raises(error, match="^(?!.*ROCm)"):
            vk.mx_cache_write(args["k"], args["v"], args["cache"], args["slots"])


def test_reads_refuse():
    for error, args in ((TypeError, (_i32(4),)), (ValueError, (_i64(4)[None],)), (TypeError, (_i64(4), torch.float64)),
                        (TypeError, ([0, 1],))):
        with pytest.raises(error, match="^(?!.*ROCm)"):
            vk.mx_cache_read(_cache(), *args)


@pytest.mark.parametrize("error,kw", [
    (TypeError, dict(q=X.double())), (ValueError, dict(q=torch.zeros(5, 3, 64))), (ValueError, dict(q=torch.zeros(5, 0, 64))),
    (ValueError, dict(q=torch.zeros(5, 2, 128))), (ValueError, dict(q=X[0])),
    (TypeError, dict(block_table=_i32(5, 2).long())), (ValueError, dict(block_table=_i32(5))),
    (TypeError, dict(lengths=_i32(5).long())), (ValueError, dict(lengths=_i32(4))),
    (ValueError, dict(block_table=_i32(4, 2), lengths=_i32(4))),          # 5 rows, 4 sequences, no q_starts
    (TypeError, dict(q_starts=_i32(6).long())), (ValueError, dict(q_starts=_i32(5))),
    (ValueError, dict(scale=float("nan"))), (ValueError, dict(scale=float("inf"))),
])
def test_attention_refuses(error, kw):
    args = dict(q=X, cache=_cache(), block_table=_i32(5, 2), lengths=_i32(5))
    args.update(kw)
    with pytest.raises(error, match="^(?!.*ROCm)"):
        vk.mx_cache_attention(**args)


def _write(lib, **kw):
    a = dict(q=None, k=16, v=32, q_out=None, cos_sin=None, positions=None, slots=48, kc=64, ks=80, vc=96, vs=112,
             tokens=4, q_heads=0, kv_heads=2, head_dim=64, q_t=0, q_h=0, k_t=128, k_h=64, v_t=128, v_h=64,
             max_pos=0, pages=3, page_size=16, dtype=2, fmt=1, stream=None)
    a.update(kw)
    return lib.velograd_mx_cache_write(*a.values())


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dtype=5), -2, "unsupported dtype"), (dict(fmt=2), -1, "mx_format"), (dict(head_dim=96), -1, "head_dim"),
    (dict(page_size=48), -1, "page_size"), (dict(page_size=8), -1, "page_size"), (dict(kv_heads=0), -1, "cache shape"),
    (dict(pages=-1), -1, "cache shape"), (dict(tokens=-1), -1, "invalid shape"), (dict(q_heads=2), -1, "invalid shape"),
    (dict(k=None), -1, "NULL"), (dict(slots=None), -1, "NULL"), (dict(kc=None), -1, "NULL"),
    (dict(positions=16), -1, "NULL"), (dict(positions=16, cos_sin=16, q_heads=2), -1, "NULL"),
    (dict(kc=72), -1, "aligned"), (dict(positions=16, cos_sin=16, q_heads=2, q=16, q_out=24), -1, "aligned"),
    (dict(positions=16, cos_sin=16, max_pos=-1), -1, "max_positions"), (dict(tokens=1 << 40), -1, "grid limit"),
])
def test_write_abi_errors(lib, kw, code, msg):
    assert _write(lib, **kw) == code
    assert msg in _lib.last_error()


def _read(lib, **kw):
    a = dict(kc=64, ks=80, vc=96, vs=112, slots=16, k=128, v=144, tokens=4, kv_heads=2, head_dim=64, pages=3,
             page_size=16, dtype=2, fmt=1, stream=None)
    a.update(kw)
    return lib.velograd_mx_cache_read(*a.values())


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dtype=5), -2, "unsupported dtype"), (dict(fmt=-1), -1, "mx_format"), (dict(head_dim=0), -1, "head_dim"),
    (dict(page_size=0), -1, "page_size"), (dict(tokens=-4), -1, "invalid shape"), (dict(v=None), -1, "NULL"),
    (dict(slots=None), -1, "NULL"), (dict(k=129), -1, "aligned"), (dict(vs=111), -1, "aligned"),
    (dict(tokens=1 << 50), -1, "grid limit"),
])
def test_read_abi_errors(lib, kw, code, msg):
    assert _read(lib, **kw) == code
    assert msg in _lib.last_error()


def _attention(lib, **kw):
    a = dict(q=16, kc=64, ks=80, vc=96, vs=112, table=16, lengths=16, starts=None, out=128, lse=None, ws=None, ws_bytes=0,
             q_tokens=4, sequences=4, q_heads=4, kv_heads=2, head_dim=64, q_t=256, q_h=64, table_stride=2, table_width=2,
             pages=3, page_size=16, scale=0.1, causal=1, dtype=2, fmt=1, stream=None)
    a.update(kw)
    return lib.velograd_mx_cache_attention(*a.values())


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dtype=5), -2, "unsupported dtype"), (dict(fmt=7), -1, "mx_format"), (dict(head_dim=32), -1, "head_dim"),
    (dict(q_heads=3), -1, "invalid shape"), (dict(q_heads=0), -1, "invalid shape"), (dict(q_tokens=5), -1, "q_starts"),
    (dict(q_tokens=-1, starts=16), -1, "invalid shape"), (dict(table_width=1 << 40), -1, "too long"),
    (dict(q_tokens=1 << 31, sequences=1 << 31), -1, "too many"), (dict(scale=float("nan")), -1, "scale"),
    (dict(q=None), -1, "NULL"), (dict(out=None), -1, "NULL"), (dict(lengths=None), -1, "NULL"),
    (dict(table=None), -1, "NULL"), (dict(vc=None), -1, "NULL"), (dict(out=136), -1, "aligned"),
    (dict(ks=81), -1, "aligned"),
])
def test_attention_abi_errors(lib, kw, code, msg):
    assert _attention(lib, **kw) == code
    assert msg in _lib.last_error()


def test_no_tokens_is_a_no_op(lib):
    assert _write(lib, tokens=0, k=None) == 0
    assert _read(lib, tokens=0, k=None) == 0
    assert _attention(lib, q_tokens=0, sequences=0, q=None) == 0
    assert _lib.last_error() == ""


def test_workspace_of_bad_arguments_is_zero(lib):
    f = lib.velograd_mx_cache_attention_workspace_bytes
    assert f(4, 4, 3, 2, 64, 2, 16, 0, 2, 1, 0) == 0
    assert f(4, 4, 4, 2, 65, 2, 16, 0, 2, 1, 0) == 0
    assert f(4, 5, 4, 2, 64, 2, 16, 0, 2, 1, 0) == 0
    assert f(4, 4, 4, 2, 64, 2, 16, 0, 9, 1, 0) == 0
    assert f(4, 4, 4, 2, 64, 2, 16, 0, 2, 9, 0) == 0
