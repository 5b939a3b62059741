"""The MX cache on the GPU: writing (with and without rotation) and reading byte for byte against the
oracle's quantiser, attention against 64 bits with a bound counted term by term (tests/_mx_cache.py)."""

import sys

import numpy as np
import pytest
import torch

from tests import _mx_cache as R
from velograd_amd import _lib
from velograd_amd import kernels as vk

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# Half a step of each type, and the rounding of the probabilities that the kernel documents: bf16 parts,
# each off by at most 2^-8 of what the parts before leave; two for 2-byte outputs, three for float32.
OUT_EPS = {t: torch.finfo(t).eps / 2 for t in DTYPES.values()}
P_EPS = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -16, torch.float32: 2.0 ** -24}
# Of chunks: one part for bf16.
CHUNK_P_EPS = {**P_EPS, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(autouse=True, params=["fast path", "general path"])
def _path(request, monkeypatch):
    """Every test through the C++ fast path and without it."""
    if request.param == "general path":
        monkeypatch.setattr(_lib, "fastpath", lambda: None)
    else:
        assert _lib.fastpath() is not None


def _say(msg):
    print(msg, flush=True)


def _randn(rng, shape, dtype):
    return torch.from_numpy(rng.standard_normal(shape, dtype=np.float32)).to("cuda", dtype)


def _f32(t):
    return t.float().cpu().numpy()


def _dirty(pages, page, heads, dim, fmt, rng):
    """A cache of leftovers: any code, any scale, NaN among them."""
    size = dim // 2 if fmt == "e2m1" else dim
    parts = []
    for _ in range(2):
        parts.append(rng.integers(0, 256, (pages, heads, page, size), dtype=np.uint8))
        s = rng.integers(100, 150, (pages, heads, dim // 32, page), dtype=np.uint8)
        s[rng.random(s.shape) < 0.3] = 255
        parts.append(s)
    return parts


def _same_bytes(cache, parts, label):
    for name, got, want in zip(("k_codes", "k_scales", "v_codes", "v_scales"), R.as_bytes(cache), parts):
        bad = np.argwhere(got != want)
        assert len(bad) == 0, (label, name, len(bad), bad[:4])


WRITE = [
    # dtype, fmt, dim, kv heads, page, pages, tokens
    ("bf16", "e2m1", 128, 8, 16, 9, 1),
    ("bf16", "e2m1", 128, 2, 64, 5, 131),
    ("bf16", "e4m3", 64, 3, 16, 40, 500),
    ("fp16", "e2m1", 256, 1, 32, 11, 77),
    ("fp16", "e4m3", 128, 5, 128, 3, 33),
    ("fp32", "e2m1", 64, 4, 16, 7, 64),
    ("fp32", "e4m3", 256, 2, 256, 2, 65),
]


@pytest.mark.parametrize("dtype,fmt,dim,heads,page,pages,tokens", WRITE)
def test_write_and_read(dtype, fmt, dim, heads, page, pages, tokens):
    _say(f"write {dtype} {fmt} dim {dim} heads {heads} page {page} tokens {tokens}")
    rng = np.random.default_rng(dim + tokens)
    dt = DTYPES[dtype]
    # k and v are slices of one projection that starts at an odd element, so nothing is aligned
    flat = _randn(rng, tokens * (3 * heads * dim) + 1, dt)
    x = flat[1:].view(tokens, 3 * heads, dim)
    k, v = x[:, heads:2 * heads], x[:, 2 * heads:]
    parts = _dirty(pages, page, heads, dim, fmt, rng)
    cache = R.from_bytes(parts, fmt, "cuda")
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    slots[tokens // 2:tokens // 2 + tokens // 5] = -1
    if tokens > 2:
        slots[-1] = pages * page          # one past the end
        slots[-2] = -(1 << 40)
    s = torch.from_numpy(slots).cuda()
    vk.mx_cache_write(k, v, cache, s)
    R.write(parts, _f32(k), _f32(v), slots, page, fmt)
    _same_bytes(cache, parts, "write")
    ok = (slots >= 0) & (slots < pages * page)
    at = np.where(ok, slots, 0)
    for out in (torch.float32, torch.bfloat16, torch.float16):
        kr, vr = vk.mx_cache_read(cache, s, out)
        for got, codes, scales in ((kr, parts[0], parts[1]), (vr, parts[2], parts[3])):
            want = R.values(codes[at // page, :, at % page], scales[at // page, :, :, at % page], fmt)
            want[~ok] = 0.0
            want = torch.from_numpy(want).to(out)
            assert got.dtype == out and got.shape == (tokens, heads, dim)
            assert torch.equal(got.cpu(), want), out
    # the leftovers (NaN blocks, the range's ends) in any order, and the same slot twice
    every = torch.from_numpy(rng.integers(0, pages * page, 50)).cuda()
    kr, vr = vk.mx_cache_read(cache, every, torch.float32)
    e = every.cpu().numpy()
    for got, codes, scales in ((kr, parts[0], parts[1]), (vr, parts[2], parts[3])):
        want = R.values(codes[e // page, :, e % page], scales[e // page, :, :, e % page], fmt)
        assert np.array_equal(_f32(got), want.astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
def test_write_special_blocks(fmt):
    _say(f"write special blocks {fmt}")
    rng = np.random.default_rng(3)
    k = rng.standard_normal((8, 2, 64), dtype=np.float32)
    k[0] = 0.0
    k[1] *= 1e-40                      # subnormal blocks
    k[2, 0, 5] = np.nan
    k[3, 1, 40] = np.inf
    k[4, 0, 0] = 3.4e38
    k[5] *= 1e-30
    k[6, 0, :32] = -0.0
    k[7] = np.float32(2.0) ** rng.integers(-126, 127, (2, 64)) * 1.75
    cache = vk.mx_cache(2, 16, 2, 64, fmt)
    parts = R.as_bytes(cache)
    slots = np.array([0, 3, 17, 31, 5, 16, 9, 8], dtype=np.int64)
    vk.mx_cache_write(torch.from_numpy(k).cuda(), torch.from_numpy(k[::-1].copy()).cuda(), cache,
                      torch.from_numpy(slots).cuda())
    R.write(parts, k, k[::-1], slots, 16, fmt)
    _same_bytes(cache, parts, "special")
    kr, _ = vk.mx_cache_read(cache, torch.from_numpy(slots).cuda(), torch.float32)
    kr = _f32(kr)
    assert np.isnan(kr[2, 0, :32]).all() and np.isfinite(kr[2, 0, 32:]).all()
    assert np.isnan(kr[3, 1, 32:]).all() and np.isfinite(kr[3, 1, :32]).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("fmt,dim", [("e2m1", 128), ("e4m3", 64), ("e2m1", 256)])
def test_rope_write(dtype, fmt, dim):
    _say(f"rope write {dtype} {fmt} {dim}")
    rng = np.random.default_rng(dim)
    dt = DTYPES[dtype]
    tokens, heads, kv, page, pages = 70, 6, 2, 32, 4
    x = _randn(rng, (tokens, heads + 2 * kv, dim), dt)
    q, k, v = x.split([heads, kv, kv], 1)
    table = vk.rope_table(5000, dim, 500000.0)
    assert table.shape == (5000, dim) and table.dtype == torch.float32
    j = np.arange(dim // 2)
    angle = 4999.0 * 500000.0 ** (-2.0 * j / dim)
    # the table's values are rounded once from 64 bits (whose own angle is good to 4999 * 2^-51)
    assert np.abs(_f32(table)[4999] - np.concatenate((np.cos(angle), np.sin(angle)))).max() <= 2.0 ** -24
    positions = rng.integers(0, 5000, tokens)
    positions[7], positions[8] = -1, 5000
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    slots[11] = -1
    cache = vk.mx_cache(pages, page, kv, dim, fmt)
    parts = R.as_bytes(cache)
    q_rot = vk.rope_mx_cache_write(q, k, v, table, torch.from_numpy(positions).cuda(), cache,
                                   torch.from_numpy(slots).cuda())
    cs = np.concatenate((_f32(table), np.full((1, dim), np.nan, np.float32)))
    pos = np.where((positions >= 0) & (positions < 5000), positions, 5000)
    want = torch.from_numpy(R.rotate(_f32(q), cs, pos)).to(dt)
    assert q_rot.dtype == dt and q_rot.shape == q.shape and q_rot.is_contiguous()
    assert np.array_equal(_f32(q_rot), want.float().numpy(), equal_nan=True)
    assert np.isnan(_f32(q_rot)[[7, 8]]).all() and np.isfinite(_f32(q_rot)[9:]).all()
    k_rot = torch.from_numpy(R.rotate(_f32(k), cs, pos)).to(dt).float().numpy()
    R.write(parts, k_rot, _f32(v), slots, page, fmt)
    _same_bytes(cache, parts, "rope")
    # without queries
    again = vk.mx_cache(pages, page, kv, dim, fmt)
    assert vk.rope_mx_cache_write(None, k, v, table, torch.from_numpy(positions).cuda(), again,
                                  torch.from_numpy(slots).cuda()) is None
    _same_bytes(again, parts, "rope without q")


def _setup(rng, dt, fmt, dim, heads, kv, page, lengths, fresh, pad, width_extra=1):
    """Sequences written into scattered pages of a cache full of leftovers."""
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + 3
    order = rng.permutation(pages)
    width = max(need, default=0) + width_extra
    table = rng.integers(-5, pages + 5, (len(lengths), width)).astype(np.int32)   # past the end: anything
    at = 0
    parts = _dirty(pages, page, kv, dim, fmt, rng)
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
        if lengths[b]:
            t = np.arange(lengths[b])
            slots = table[b, t // page].astype(np.int64) * page + t % page
            R.write(parts, rng.standard_normal((lengths[b], kv, dim), dtype=np.float32) *
                    np.exp(0.5 * rng.standard_normal(dim, dtype=np.float32)),
                    rng.standard_normal((lengths[b], kv, dim), dtype=np.float32), slots, page, fmt)
    starts = np.concatenate(([0], np.cumsum(fresh))).astype(np.int32) if fresh is not None else None
    tokens = (len(lengths) if fresh is None else int(sum(fresh))) + pad
    q = _randn(rng, (tokens, heads + 1, dim), dt)[:, 1:]
    return parts, table, starts, q


@pytest.fixture(params=["short table", "long table"])
def table_room(request, monkeypatch):
    """A table with room for few keys lets few rows take one launch, one with room for many is split."""
    monkeypatch.setattr(sys.modules[__name__], "LONG_TABLE", request.param == "long table")


LONG_TABLE = False


def _attend(q, parts, table, lengths, starts, fmt, **kw):
    cache = R.from_bytes(parts, fmt, "cuda")
    if LONG_TABLE:
        table = np.pad(table, ((0, 0), (0, (1 << 20) // parts[0].shape[2])), constant_values=-9)
    t = torch.from_numpy(table).cuda()
    ln = torch.tensor(lengths, dtype=torch.int32).cuda()
    st = None if starts is None else torch.from_numpy(np.asarray(starts, dtype=np.int32)).cuda()
    return vk.mx_cache_attention(q, cache, t, ln, st, return_lse=True, **kw)


def _check(got, q, parts, table, lengths, starts, page, fmt, scale=None, causal=True, p_eps=None):
    out, lse = got
    dim = q.shape[-1]
    scale = dim ** -0.5 if scale is None else scale
    want, wlse, off, lse_off = R.attention(q.double().cpu().numpy(), parts, table, lengths, starts, page, fmt,
                                           scale, causal, OUT_EPS[q.dtype], P_EPS[q.dtype] if p_eps is None else p_eps)
    assert out.dtype == q.dtype and out.shape == q.shape and lse.dtype == torch.float32
    o, s = out.double().cpu().numpy(), lse.double().cpu().numpy()
    empty = np.isneginf(wlse)
    assert np.array_equal(empty, np.isneginf(s))
    assert (o[empty] == 0).all()
    # outputs under the type's normal range round to its smallest step
    floor = torch.finfo(q.dtype).tiny * OUT_EPS[q.dtype]
    bad = np.argwhere(np.abs(o - want) > off + floor)
    assert len(bad) == 0, (len(bad), bad[0], o[tuple(bad[0])], want[tuple(bad[0])], off[tuple(bad[0])])
    s, wlse = np.where(empty, 0.0, s), np.where(empty, 0.0, wlse)
    bad = np.argwhere(np.abs(s - wlse) > lse_off)
    assert len(bad) == 0, (len(bad), bad[0], s[tuple(bad[0])], wlse[tuple(bad[0])], lse_off[tuple(bad[0])])


ATTENTION = [
    # dtype, fmt, dim, heads, kv heads, page, lengths, new tokens (None: one each), padding rows
    ("bf16", "e2m1", 128, 8, 2, 16, [1], None, 0),
    ("bf16", "e2m1", 128, 32, 8, 16, [2, 15, 16, 17, 31, 32, 33, 500], None, 0),
    ("bf16", "e2m1", 64, 6, 3, 64, [0, 129, 0, 64], None, 0),
    ("fp16", "e4m3", 256, 4, 1, 32, [700, 3], None, 0),
    ("fp32", "e2m1", 128, 5, 1, 16, [257, 31, 1], None, 0),
    ("fp32", "e4m3", 64, 4, 4, 256, [300, 1], None, 0),
    ("bf16", "e4m3", 128, 40, 1, 16, [100, 45], None, 0),         # more rows than one tile
    ("bf16", "e2m1", 128, 160, 1, 16, [100, 45], None, 0),
    ("bf16", "e2m1", 128, 8, 2, 16, [40, 5, 300], [3, 5, 8], 0),  # drafted tokens
    ("bf16", "e2m1", 128, 4, 1, 64, [200], [200], 0),             # a whole prompt
    ("fp16", "e2m1", 64, 8, 4, 16, [333, 70, 9, 0], [150, 1, 9, 2], 5),
    ("fp32", "e4m3", 128, 2, 1, 32, [90, 65], [64, 2], 1),
    ("fp32", "e2m1", 256, 4, 2, 16, [90, 31], [33, 31], 0),
    ("bf16", "e4m3", 256, 3, 1, 16, [10, 50], [20, 50], 3),       # more new tokens than held: empty rows
    ("bf16", "e2m1", 128, 16, 2, 16, [3000], None, 0),            # split over the keys
    ("fp16", "e2m1", 128, 16, 2, 128, [2500, 1, 900], [2, 1, 7], 2),
    ("fp32", "e2m1", 64, 8, 1, 16, [4100, 5], None, 0),
    # many sequences, of very unequal lengths
    ("bf16", "e2m1", 64, 2, 1, 16, [1 + 7 * i % 50 + (1500 if i % 67 == 66 else 0) for i in range(300)], None, 0),
    ("fp16", "e4m3", 64, 4, 2, 16, [9 * i % 40 + (700 if i % 97 == 96 else 0) for i in range(200)],
     [i % 3 + (30 if i % 50 == 7 else 0) for i in range(200)], 17),
    ("fp32", "e2m1", 128, 3, 3, 32, [5 + i % 2 for i in range(130)], [1] * 130, 0),
]


@pytest.mark.usefixtures("table_room")
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,fmt,dim,heads,kv,page,lengths,fresh,pad", ATTENTION)
def test_attention(dtype, fmt, dim, heads, kv, page, lengths, fresh, pad, causal):
    _say(f"attention {dtype} {fmt} dim {dim} {heads}/{kv} page {page} {lengths} {fresh} pad {pad} causal {causal}")
    rng = np.random.default_rng(sum(lengths) + dim)
    parts, table, starts, q = _setup(rng, DTYPES[dtype], fmt, dim, heads, kv, page, lengths, fresh, pad)
    got = _attend(q, parts, table, lengths, starts, fmt, causal=causal)
    _check(got, q, parts, table, lengths, starts, page, fmt, causal=causal)
    # the same call gives the same bits
    again = _attend(q, parts, table, lengths, starts, fmt, causal=causal)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


CHUNKS = [
    # enough rows for the kernel that takes 64 rows of a sequence a wave, others and padding beside them:
    # dtype, fmt, dim, heads, kv heads, page, lengths, new tokens, padding rows
    ("bf16", "e2m1", 64, 32, 8, 16, [2100], [2060], 0),
    ("bf16", "e2m1", 128, 16, 2, 64, [1500, 40, 0, 3000, 333], [1500, 1, 3, 2400, 250], 70),
    ("bf16", "e4m3", 256, 24, 3, 32, [1400], [1399], 1),
    ("fp16", "e2m1", 128, 30, 6, 16, [1300, 17], [1280, 2], 300),
    ("fp32", "e4m3", 64, 40, 8, 128, [900, 10], [880, 20], 0),
    ("fp32", "e2m1", 128, 32, 32, 16, [600, 700], [500, 600], 3),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,fmt,dim,heads,kv,page,lengths,fresh,pad", CHUNKS)
def test_attention_of_chunks(dtype, fmt, dim, heads, kv, page, lengths, fresh, pad, causal):
    _say(f"chunks {dtype} {fmt} dim {dim} {heads}/{kv} page {page} {lengths} {fresh} pad {pad} causal {causal}")
    rng = np.random.default_rng(sum(lengths) + dim)
    parts, table, starts, q = _setup(rng, DTYPES[dtype], fmt, dim, heads, kv, page, lengths, fresh, pad)
    got = _attend(q, parts, table, lengths, starts, fmt, causal=causal)
    _check(got, q, parts, table, lengths, starts, page, fmt, causal=causal, p_eps=CHUNK_P_EPS[DTYPES[dtype]])
    again = _attend(q, parts, table, lengths, starts, fmt, causal=causal)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_chunks_keep_nan_values_from_rows_that_do_not_see_them():
    _say("chunks NaN")
    rng = np.random.default_rng(17)
    parts, table, starts, q = _setup(rng, torch.bfloat16, "e2m1", 64, 32, 1, 16, [2200], [2100], 0)
    clean = _attend(q, parts, table, [2200], starts, "e2m1")
    for t in (50, 1000):
        parts[3][table[0, t // 16], 0, 1, t % 16] = 255          # dims 32..63
    out, lse = _attend(q, parts, table, [2200], starts, "e2m1")
    assert torch.isnan(out[..., 32:]).all()                       # every row sees key 50
    assert torch.equal(out[..., :32], clean[0][..., :32]) and torch.equal(lse, clean[1])
    parts[3][table[0, 50 // 16], 0, 1, 50 % 16] = 127
    parts[2][table[0, 50 // 16], 0, 50 % 16] = 0
    clean = _attend(q, parts, table, [2200], starts, "e2m1")
    out, lse = _attend(q, parts, table, [2200], starts, "e2m1")
    first = 1000 - 100                                            # row i sees keys up to 100 + i
    assert torch.isnan(out[first:, :, 32:]).all() and not torch.isnan(out[:first]).any()
    assert torch.equal(out[..., :32], clean[0][..., :32])


@pytest.mark.parametrize("dtype,dim,heads", [("bf16", 128, 16), ("fp16", 64, 24), ("fp32", 256, 16)])
def test_chunks_with_missing_pages_and_nan_codes(dtype, dim, heads):
    """From a missing page on, a chunk's steps are masked; e4m3 has NaN codes of single elements."""
    _say(f"chunks bad pages {dtype} {dim}")
    rng = np.random.default_rng(dim)
    lengths, fresh = [2500, 31, 400], [2450, 2, 390]
    parts, table, starts, q = _setup(rng, DTYPES[dtype], "e4m3", dim, heads, 1, 16, lengths, fresh, 3)
    table[0, 3], table[0, 60], table[0, 101:103], table[2, :2] = -1, parts[0].shape[0], 1 << 30, -(1 << 31)
    got = _attend(q, parts, table, lengths, starts, "e4m3")
    _check(got, q, parts, table, lengths, starts, 16, "e4m3", p_eps=CHUNK_P_EPS[DTYPES[dtype]])
    at = 1234
    parts[2][table[0, at // 16], 0, at % 16, 5] = 0xff
    out, lse = _attend(q, parts, table, lengths, starts, "e4m3")
    first = at - (2500 - 2450)
    assert torch.isnan(out[first:2450, :, 5]).all() and torch.equal(lse, got[1])
    out[first:2450, :, 5] = got[0][first:2450, :, 5]
    assert torch.equal(out, got[0])
    parts[0][table[0, at // 16], 0, at % 16, 7] = 0x7f                  # a key: whole rows
    out, lse = _attend(q, parts, table, lengths, starts, "e4m3")
    assert torch.isnan(out[first:2450]).all() and torch.isnan(lse[first:2450]).all()
    assert torch.equal(out[:first], got[0][:first]) and torch.equal(out[2450:], got[0][2450:])


@pytest.mark.parametrize("scale", [0.0, 2.0, -0.3])
def test_chunks_scales(scale):
    _say(f"chunks scale {scale}")
    rng = np.random.default_rng(41)
    parts, table, starts, q = _setup(rng, torch.bfloat16, "e2m1", 64, 32, 2, 32, [1300, 70], [1290, 5], 0)
    got = _attend(q, parts, table, [1300, 70], starts, "e2m1", scale=scale)
    _check(got, q, parts, table, [1300, 70], starts, 32, "e2m1", scale=scale, p_eps=CHUNK_P_EPS[torch.bfloat16])


@pytest.mark.usefixtures("table_room")
@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3])
def test_attention_scales(scale):
    _say(f"attention scale {scale}")
    rng = np.random.default_rng(5)
    parts, table, starts, q = _setup(rng, torch.bfloat16, "e2m1", 128, 8, 2, 16, [90, 33], [3, 1], 0)
    got = _attend(q, parts, table, [90, 33], starts, "e2m1", scale=scale)
    _check(got, q, parts, table, [90, 33], starts, 16, "e2m1", scale=scale)


@pytest.mark.usefixtures("table_room")
def test_attention_skips_pages_outside_the_cache():
    _say("attention bad pages")
    rng = np.random.default_rng(6)
    lengths, fresh = [100, 64, 200], [1, 20, 2]
    parts, table, starts, q = _setup(rng, torch.bfloat16, "e2m1", 128, 8, 2, 16, lengths, fresh, 0)
    table[0, 2], table[0, 6] = -1, parts[0].shape[0]
    table[1, :4] = 1 << 30                       # nothing left to see
    table[2, 0] = -(1 << 31)
    got = _attend(q, parts, table, lengths, starts, "e2m1")
    _check(got, q, parts, table, lengths, starts, 16, "e2m1")
    assert (got[0][1:21] == 0).all() and torch.isneginf(got[1][1:21]).all()


@pytest.mark.usefixtures("table_room")
@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("fresh", [[40], [1]])
def test_attention_nan_keys_and_values_reach_only_rows_that_see_them(fmt, fresh):
    _say(f"attention NaN {fmt} {fresh}")
    rng = np.random.default_rng(7)
    parts, table, starts, q = _setup(rng, torch.bfloat16, fmt, 128, 4, 1, 16, [80], fresh, 0)
    clean = _attend(q, parts, table, [80], starts, fmt)
    t = 70
    page = table[0, t // 16]
    parts[3][page, 0, 1, t % 16] = 255           # dims 32..63 of one value
    out, lse = _attend(q, parts, table, [80], starts, fmt)
    first = 80 - fresh[0]                        # row i sees keys up to first + i
    for i in range(fresh[0]):
        if first + i < t:
            assert torch.equal(out[i], clean[0][i]), i
        else:
            assert torch.isnan(out[i, :, 32:64]).all(), i
            assert torch.equal(out[i, :, :32], clean[0][i, :, :32]), i
            assert torch.equal(out[i, :, 64:], clean[0][i, :, 64:]), i
    assert torch.equal(lse, clean[1])
    parts[1][page, 0, 0, t % 16] = 255           # and a part of the key: every score of it is NaN
    out, lse = _attend(q, parts, table, [80], starts, fmt)
    for i in range(fresh[0]):
        if first + i < t:
            assert torch.equal(out[i], clean[0][i]) and torch.equal(lse[i], clean[1][i]), i
        else:
            assert torch.isnan(out[i]).all() and torch.isnan(lse[i]).all(), i


@pytest.mark.usefixtures("table_room")
def test_attention_nan_and_infinite_queries_stay_in_their_row():
    _say("attention NaN queries")
    rng = np.random.default_rng(8)
    for dtype in DTYPES.values():
        parts, table, starts, q = _setup(rng, dtype, "e2m1", 128, 4, 2, 16, [50], [6], 0)
        clean = _attend(q, parts, table, [50], starts, "e2m1")
        q = q.clone()
        q[2, 1, 100] = float("nan")
        q[4, 3, 0] = float("inf")
        out, lse = _attend(q, parts, table, [50], starts, "e2m1")
        bad = torch.zeros(6, 4, dtype=torch.bool, device="cuda")
        bad[2, 1] = bad[4, 3] = True
        assert torch.isnan(out[bad]).all() and torch.isnan(lse[2, 1])
        assert torch.equal(out[~bad], clean[0][~bad]) and torch.equal(lse[~bad], clean[1][~bad])


@pytest.mark.usefixtures("table_room")
def test_attention_rows_of_no_sequence():
    _say("attention rows of no sequence")
    rng = np.random.default_rng(9)
    parts, table, starts, q = _setup(rng, torch.bfloat16, "e2m1", 64, 4, 2, 16, [40, 60], [4, 3], 10)
    starts = starts + 3                          # three rows before the first sequence, seven behind the last
    out, lse = _attend(q, parts, table, [40, 60], starts, "e2m1")
    _check((out, lse), q, parts, table, [40, 60], starts, 16, "e2m1")
    assert (out[:3] == 0).all() and (out[10:] == 0).all() and torch.isneginf(lse[10:]).all()
    # no sequence, no page, no width
    cache = vk.mx_cache(0, 16, 2, 64)
    none = torch.zeros(0, 4, dtype=torch.int32, device="cuda")
    out = vk.mx_cache_attention(q, cache, none, none[:, 0].contiguous(), torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert (out == 0).all()
    for width in (0, 3):
        table = torch.zeros(len(q), width, dtype=torch.int32, device="cuda")
        out = vk.mx_cache_attention(q, cache, table, torch.full((len(q),), 7, dtype=torch.int32, device="cuda"))
        assert (out == 0).all()


def test_lengths_past_the_table_and_below_zero_are_clamped():
    _say("attention clamped lengths")
    rng = np.random.default_rng(10)
    parts, table, starts, q = _setup(rng, torch.bfloat16, "e2m1", 128, 4, 2, 16, [64, 64, 64], None, 0, 0)
    want = _attend(q, parts, table, [64, 64, 0], starts, "e2m1")
    got = _attend(q, parts, table, [1 << 30, 65, -7], starts, "e2m1")
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_falling_starts_leave_the_buffers_alone():
    """Outside the contract: rows are unspecified, but nothing past the buffers is touched."""
    _say("falling starts")
    rng = np.random.default_rng(31)
    lengths = [300 + 5 * i for i in range(90)]
    for tokens, heads in ((180, 8), (2100, 32)):              # the step kernel's call, the chunk kernel's
        fresh = [tokens // 90] * 90
        fresh[0] += tokens - sum(fresh)
        parts, table, starts, q = _setup(rng, torch.bfloat16, "e2m1", 64, heads, 2, 16, lengths, fresh, 0, 70000)
        want = _attend(q, parts, table, lengths, starts, "e2m1")
        bad = starts.copy()
        bad[1::2], bad[2::2] = tokens, 0
        out, lse = _attend(q, parts, table, lengths, bad, "e2m1")
        torch.cuda.synchronize()
        assert out.shape == q.shape and lse.shape == q.shape[:2]
        again = _attend(q, parts, table, lengths, starts, "e2m1")
        assert torch.equal(want[0], again[0]) and torch.equal(want[1], again[1])


def test_empty_calls():
    _say("empty calls")
    cache = vk.mx_cache(2, 16, 2, 64, "e4m3")
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    x = torch.zeros(0, 2, 64, device="cuda")
    vk.mx_cache_write(x, x, cache, none)
    assert vk.rope_mx_cache_write(x, x, x, vk.rope_table(0, 64), none, cache, none).shape == (0, 2, 64)
    k, v = vk.mx_cache_read(cache, none)
    assert k.shape == v.shape == (0, 2, 64)
    out = vk.mx_cache_attention(x, cache, torch.zeros(0, 1, dtype=torch.int32, device="cuda"), none.int())
    assert out.shape == (0, 2, 64)


def test_generation_through_the_cache():
    """A prompt, then single tokens, each rotated and written, then attended to: as one would serve."""
    _say("generation")
    rng = np.random.default_rng(11)
    heads, kv, dim, page, fmt = 8, 2, 128, 16, "e2m1"
    prompts, steps = [37, 5, 18], 20
    cos_sin = vk.rope_table(100, dim)
    pages = 20
    cache = vk.mx_cache(pages, page, kv, dim, fmt)
    parts = R.as_bytes(cache)
    table = rng.permutation(pages)[:3 * 4].reshape(3, 4).astype(np.int32)
    held = [0, 0, 0]
    for step in range(steps):
        fresh = prompts if step == 0 else [1, 1, 1]
        held = [h + n for h, n in zip(held, fresh)]
        pos = np.concatenate([np.arange(h - n, h) for h, n in zip(held, fresh)])
        seq = np.repeat(np.arange(3), fresh)
        slots = table[seq, pos // page].astype(np.int64) * page + pos % page
        x = _randn(rng, (len(pos), heads + 2 * kv, dim), torch.bfloat16)
        q, k, v = x.split([heads, kv, kv], 1)
        q_rot = vk.rope_mx_cache_write(q, k, v, cos_sin, torch.from_numpy(pos).cuda(), cache,
                                       torch.from_numpy(slots).cuda())
        starts = np.concatenate(([0], np.cumsum(fresh))).astype(np.int32) if step == 0 else None
        got = vk.mx_cache_attention(q_rot, cache, torch.from_numpy(table).cuda(),
                                    torch.tensor(held, dtype=torch.int32).cuda(),
                                    None if starts is None else torch.from_numpy(starts).cuda(), return_lse=True)
        rot = lambda t: torch.from_numpy(R.rotate(_f32(t), _f32(cos_sin), pos)).to(torch.bfloat16)  # noqa: E731
        assert torch.equal(q_rot.cpu(), rot(q))
        R.write(parts, rot(k).float().numpy(), _f32(v), slots, page, fmt)
        _same_bytes(cache, parts, step)
        _check(got, q_rot, parts, table, held, starts, page, fmt)


def test_split_keys_join_with_lse():
    """Attention over a sequence in two parts, joined by lse, is attention over all of it."""
    _say("join by lse")
    rng = np.random.default_rng(12)
    parts, table, _, q = _setup(rng, torch.float32, "e4m3", 64, 4, 2, 16, [160], None, 0, 0)
    whole, lse = _attend(q, parts, table, [160], None, "e4m3")
    a, la = _attend(q, parts, table[:, :6].copy(), [96], None, "e4m3")
    b, lb = _attend(q, parts, table[:, 6:].copy(), [64], None, "e4m3")
    joined = torch.logaddexp(la, lb)
    both = a * torch.exp(la - joined)[..., None] + b * torch.exp(lb - joined)[..., None]
    # float32 throughout: a few ulps of values of at most ~4, and of |lse| < 16 in the exponent
    assert (both - whole).abs().max() < 64 * 2.0 ** -24 * 4 and (joined - lse).abs().max() < 16 * 2.0 ** -22


def test_caches_past_4_gib():
    _say("a cache past 4 GiB")
    kv, dim, page, fmt = 8, 256, 256, "e4m3"
    pages = (1 << 32) // (kv * page * dim) + 40
    cache = vk.mx_cache(pages, page, kv, dim, fmt)
    assert cache.k_codes.numel() > 1 << 32
    rng = np.random.default_rng(13)
    n = 300
    k, v = _randn(rng, (n, kv, dim), torch.bfloat16), _randn(rng, (n, kv, dim), torch.bfloat16)
    table = torch.tensor([[pages - 1, pages - 20]], dtype=torch.int32, device="cuda")
    t = torch.arange(n, device="cuda")
    slots = table[0, t // page].long() * page + t % page
    vk.mx_cache_write(k, v, cache, slots)
    kr, vr = vk.mx_cache_read(cache, slots, torch.float32)
    small = vk.mx_cache(2, page, kv, dim, fmt)
    vk.mx_cache_write(k, v, small, t)
    ks, vs = vk.mx_cache_read(small, t, torch.float32)
    assert torch.equal(kr, ks) and torch.equal(vr, vs)
    assert int(cache.k_codes[:40].view(torch.uint8).count_nonzero()) == 0
    q = _randn(rng, (1, kv, dim), torch.bfloat16)
    held = torch.tensor([n], dtype=torch.int32, device="cuda")
    out = vk.mx_cache_attention(q, cache, table, held)
    assert torch.equal(out, vk.mx_cache_attention(q, small, torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), held))


def test_a_layer_of_a_larger_allocation_and_strided_index_tensors():
    _say("layer slices, strided tables")
    rng = np.random.default_rng(14)
    parts, table, starts, q = _setup(rng, torch.bfloat16, "e2m1", 128, 4, 2, 16, [90, 33], [3, 1], 0)
    want = _attend(q, parts, table, [90, 33], starts, "e2m1")
    layers = [torch.stack([torch.from_numpy(p).cuda()] * 3) for p in parts]
    cache = tuple(t[1].view(d) for t, d in zip(layers, (torch.float4_e2m1fn_x2, torch.float8_e8m0fnu) * 2))
    wide = torch.full((2, 2 * table.shape[1]), -9, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = torch.from_numpy(table).cuda()
    ln = torch.tensor([90, 0, 33, 0], dtype=torch.int32, device="cuda")[::2]
    st = torch.from_numpy(np.repeat(starts, 2)).cuda()[::2]
    got = vk.mx_cache_attention(q, cache, wide[:, :table.shape[1]], ln, st, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # heads inside tokens, or tokens inside heads
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    got = vk.mx_cache_attention(qt, cache, wide[:, :table.shape[1]], ln, st)
    assert torch.equal(got, want[0])


@pytest.mark.parametrize("each", [200, 60])   # pages of a sequence: split over the keys, in one launch
def test_captured_and_replayed_between_eager_calls(each):
    _say(f"graphs {each}")
    rng = np.random.default_rng(15)
    heads, kv, dim, page, fmt, seqs = 8, 2, 128, 16, "e2m1", 3
    cos_sin = vk.rope_table(4000, dim)
    pages = 3 * each
    cache = vk.mx_cache(pages, page, kv, dim, fmt)
    eager = vk.mx_cache(pages, page, kv, dim, fmt)
    base = _randn(rng, (pages * page, 2 * kv, dim), torch.bfloat16)
    for c in (cache, eager):
        vk.mx_cache_write(base[:, :kv], base[:, kv:], c, torch.arange(pages * page, device="cuda"))
    table = torch.arange(pages, device="cuda", dtype=torch.int32).view(seqs, -1)
    x = torch.zeros(seqs, heads + 2 * kv, dim, device="cuda", dtype=torch.bfloat16)
    pos = torch.zeros(seqs, device="cuda", dtype=torch.int64)
    slots = torch.zeros(seqs, device="cuda", dtype=torch.int64)
    held = torch.zeros(seqs, device="cuda", dtype=torch.int32)

    def step(c):
        q, k, v = x.split([heads, kv, kv], 1)
        q = vk.rope_mx_cache_write(q, k, v, cos_sin, pos, c, slots)
        return vk.mx_cache_attention(q, c, table, held, return_lse=True)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step(cache)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(cache))
        graphs.append(g)
    for n in range(6):
        at = [(700 * n + 1000 * i) % (each * page - 100) for i in range(seqs)]
        x.copy_(_randn(rng, x.shape, torch.bfloat16))
        pos.copy_(torch.tensor(at))
        held.copy_(torch.tensor(at, dtype=torch.int32) + 1)
        slots.copy_(table[torch.arange(seqs), torch.tensor(at, device="cuda") // page].long() * page
                    + torch.tensor(at, device="cuda") % page)
        graphs[n % 2].replay()
        want = step(eager)
        torch.cuda.synchronize()
        got = outs[n % 2]
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), n
        for a, b in zip(cache, eager):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), n


def test_chunks_captured_with_other_lengths():
    """A captured call takes its sequences' rows and lengths from device memory at each replay."""
    _say("chunks graph")
    rng = np.random.default_rng(43)
    parts, table, starts, q = _setup(rng, torch.bfloat16, "e2m1", 64, 32, 4, 16, [1500, 900, 40], [1200, 60, 20], 40)
    cache = R.from_bytes(parts, "e2m1", "cuda")
    t = torch.from_numpy(table).cuda()
    held = torch.tensor([1500, 900, 40], dtype=torch.int32, device="cuda")
    at = torch.from_numpy(starts).cuda()
    vk.mx_cache_attention(q, cache, t, held, at, return_lse=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = vk.mx_cache_attention(q, cache, t, held, at, return_lse=True)
    for new, lens in (([1200, 60, 20], [1500, 900, 40]), ([1, 1, 1], [1500, 3, 0]), ([0, 890, 30], [700, 900, 35]),
                      ([1310, 2, 0], [1400, 17, 16])):
        held.copy_(torch.tensor(lens, dtype=torch.int32))
        at.copy_(torch.tensor(np.concatenate(([0], np.cumsum(new))), dtype=torch.int32))
        graph.replay()
        want = vk.mx_cache_attention(q, cache, t, held, at, return_lse=True)
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1]), (new, lens)
        assert (out[sum(new):] == 0).all() and torch.isneginf(lse[sum(new):]).all()


def test_streams():
    _say("streams")
    rng = np.random.default_rng(16)
    parts, table, starts, q = _setup(rng, torch.bfloat16, "e2m1", 128, 8, 1, 16, [3000, 10], None, 0)
    want = _attend(q, parts, table, [3000, 10], starts, "e2m1")
    cache = R.from_bytes(parts, "e2m1", "cuda")
    t, ln = torch.from_numpy(table).cuda(), torch.tensor([3000, 10], dtype=torch.int32).cuda()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(vk.mx_cache_attention(q, cache, t, ln, return_lse=True))
    torch.cuda.synchronize()
    for out, lse in outs:
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
