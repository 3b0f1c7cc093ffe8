"""The key/value cache's calls on the CPU: what the host refuses before any
launch, and the oracle's own codes."""
import ctypes as C

import numpy as np
import pytest
import torch

from kernels_amd import kq
from tests import _kv

FAKE = 0x10000


def cache_c(**kw):
    a = dict(k=FAKE, v=FAKE, k_exp=FAKE, v_exp=FAKE, type=kq.KV_I8, n_pages=64, page=16, block=16, heads=8, head_dim=128)
    a.update(kw)
    return kq._KVCacheC(**a)


def batch_c(**kw):
    a = dict(pages=FAKE, kv_len=FAKE, q_start=FAKE, n_seq=2, max_pages=8, max_q=3, n_rows=6, max_len=100)
    a.update(kw)
    return kq._KVBatchC(**a)


def rows_c(**kw):
    a = dict(p=FAKE, row=1024, head=128)
    a.update(kw)
    return kq._KVRowsC(**a)


def attn_c(**kw):
    a = dict(q_heads=32, scale=0.1, causal=1, window=0, sinks=None)
    a.update(kw)
    return kq._KVAttnC(**a)


def write(c=None, b=None, K=None, V=None, dt=kq.F16, read=False):
    f = kq.lib().kq_kv_read if read else kq.lib().kq_kv_write
    return f(C.byref(c or cache_c()), C.byref(b or batch_c()), C.byref(K or rows_c()), C.byref(V or rows_c()), dt, None)


def size(c=None, b=None, q_heads=32):
    return kq.lib().kq_kv_attn_workspace_size(C.byref(c or cache_c()), C.byref(b or batch_c()), q_heads)


def attn(c=None, b=None, d=None, Q=None, O=None, dt=kq.F16, lse=None, ws=FAKE, n=1 << 30):
    return kq.lib().kq_kv_attn(C.byref(c or cache_c()), C.byref(b or batch_c()), C.byref(d or attn_c()),
                               C.byref(Q or rows_c(row=4096)), C.byref(O or rows_c(row=4096)), dt, lse, ws, n, None)


BAD_CACHE = [
    (dict(type=2), kq.KQ_EUNSUPPORTED), (dict(head_dim=80), kq.KQ_EUNSUPPORTED), (dict(head_dim=0), kq.KQ_EUNSUPPORTED),
    (dict(head_dim=512), kq.KQ_EUNSUPPORTED), (dict(block=8), kq.KQ_EINVAL), (dict(block=48, page=48), kq.KQ_EINVAL),
    (dict(block=512, page=512), kq.KQ_EINVAL), (dict(block=32), kq.KQ_EINVAL), (dict(page=24), kq.KQ_EINVAL),
    (dict(page=8192), kq.KQ_EINVAL), (dict(page=0), kq.KQ_EINVAL), (dict(heads=0), kq.KQ_EINVAL),
    (dict(heads=1025), kq.KQ_EINVAL), (dict(n_pages=0), kq.KQ_EINVAL), (dict(n_pages=1 << 31), kq.KQ_EINVAL)]
BAD_CACHE_P = [(dict(k=None), kq.KQ_ENULL), (dict(v=None), kq.KQ_ENULL), (dict(k_exp=None), kq.KQ_ENULL),
               (dict(v_exp=None), kq.KQ_ENULL), (dict(k=FAKE + 8), kq.KQ_EALIGN), (dict(v=FAKE + 1), kq.KQ_EALIGN)]
BAD_BATCH = [
    (dict(n_seq=0), kq.KQ_EINVAL), (dict(n_seq=65536), kq.KQ_EINVAL), (dict(max_pages=0), kq.KQ_EINVAL),
    (dict(max_q=0), kq.KQ_EINVAL), (dict(max_len=0), kq.KQ_EINVAL), (dict(max_len=0x7FFF0000), kq.KQ_EINVAL),
    (dict(n_rows=0x80000000), kq.KQ_EINVAL), (dict(max_q=0x80000000), kq.KQ_EINVAL),
    (dict(q_start=None, n_rows=5), kq.KQ_EINVAL)]
BAD_BATCH_P = [(dict(pages=None), kq.KQ_ENULL), (dict(kv_len=None), kq.KQ_ENULL), (dict(pages=FAKE + 2), kq.KQ_EALIGN),
               (dict(kv_len=FAKE + 1), kq.KQ_EALIGN), (dict(q_start=FAKE + 2), kq.KQ_EALIGN)]


@pytest.mark.parametrize("kw,status", BAD_CACHE + BAD_CACHE_P)
def test_bad_cache(kw, status):
    c = cache_c(**kw)
    assert write(c) == write(c, read=True) == attn(c) == status


@pytest.mark.parametrize("kw,status", BAD_BATCH + BAD_BATCH_P)
def test_bad_batch(kw, status):
    b = batch_c(**kw)
    assert write(b=b) == write(b=b, read=True) == attn(b=b) == status


@pytest.mark.parametrize("kw,status", [
    (dict(p=None), kq.KQ_ENULL), (dict(p=FAKE + 8), kq.KQ_EALIGN), (dict(row=-1024), kq.KQ_EINVAL),
    (dict(head=-128), kq.KQ_EINVAL), (dict(row=1028), kq.KQ_EINVAL), (dict(head=132), kq.KQ_EINVAL)])
def test_bad_rows(kw, status):
    r = rows_c(**kw)
    assert write(K=r) == write(V=r) == write(K=r, read=True) == write(V=r, read=True) == status
    r = rows_c(**dict(dict(row=4096), **kw))
    assert attn(Q=r) == attn(O=r) == status


def test_strides_of_single_rows_and_heads():
    """A stride that nothing is reached by is not looked at: such calls are refused for what follows only."""
    one = batch_c(n_seq=1, n_rows=1, max_q=1)
    assert write(cache_c(heads=1), one, rows_c(row=3, head=-5), rows_c(row=3, head=-5), dt=kq.F32) == kq.KQ_EUNSUPPORTED
    assert attn(cache_c(heads=1), one, attn_c(q_heads=1), rows_c(row=1, head=1), rows_c(row=-1, head=0), ws=None) == kq.KQ_EWORKSPACE
    assert attn(cache_c(heads=1), batch_c(), attn_c(q_heads=1), rows_c(row=1, head=1), rows_c(), ws=None) == kq.KQ_EINVAL
    assert attn(cache_c(heads=1), one, attn_c(q_heads=2), rows_c(row=1, head=1), rows_c(), ws=None) == kq.KQ_EINVAL


def test_no_rows():
    """A call of no rows, whose tensors have no address, is checked and does nothing."""
    none, r = batch_c(n_rows=0), rows_c(p=None)
    assert write(b=none, K=r, V=r) == write(b=none, K=r, V=r, read=True) == attn(b=none, Q=r, O=r) == kq.KQ_OK
    assert write(cache_c(type=3), none, r, r) == attn(b=none, Q=r, O=r, dt=kq.F32) == kq.KQ_EUNSUPPORTED
    assert attn(b=none, Q=r, O=r, ws=None) == kq.KQ_EWORKSPACE
    assert write(b=batch_c(n_rows=0, q_start=None), K=r, V=r) == kq.KQ_EINVAL


@pytest.mark.parametrize("kw", [dict(row=0), dict(head=0), dict(row=120), dict(head=64)])
def test_overlapping_outputs_are_refused(kw):
    r = rows_c(**kw)
    assert write(K=r, read=True) == write(V=r, read=True) == attn(O=r) == kq.KQ_EINVAL


def test_types():
    assert write(dt=kq.F32) == kq.KQ_EUNSUPPORTED
    assert write(dt=3) == write(dt=3, read=True) == kq.KQ_EUNSUPPORTED
    assert attn(dt=kq.F32) == kq.KQ_EUNSUPPORTED


@pytest.mark.parametrize("kw", [dict(q_heads=0), dict(q_heads=12), dict(q_heads=8 * 65), dict(scale=float("nan")),
                                dict(scale=float("inf")), dict(causal=0, window=5)])
def test_bad_attention(kw):
    assert attn(d=attn_c(**kw)) == kq.KQ_EINVAL


def test_null_structs():
    L = kq.lib()
    c, b, r, d = cache_c(), batch_c(), rows_c(row=4096), attn_c()
    assert L.kq_kv_write(None, C.byref(b), C.byref(r), C.byref(r), 0, None) == kq.KQ_ENULL
    assert L.kq_kv_read(C.byref(c), None, C.byref(r), C.byref(r), 0, None) == kq.KQ_ENULL
    assert L.kq_kv_write(C.byref(c), C.byref(b), None, C.byref(r), 0, None) == kq.KQ_ENULL
    assert L.kq_kv_attn(C.byref(c), C.byref(b), None, C.byref(r), C.byref(r), 0, None, FAKE, 1 << 30, None) == kq.KQ_ENULL
    assert L.kq_kv_attn(C.byref(c), C.byref(b), C.byref(d), C.byref(r), None, 0, None, FAKE, 1 << 30, None) == kq.KQ_ENULL
    assert L.kq_kv_attn_workspace_size(None, C.byref(b), 32) == 0


def test_attention_pointers_and_workspace():
    assert attn(lse=FAKE + 2) == attn(d=attn_c(sinks=FAKE + 1)) == kq.KQ_EALIGN
    b = batch_c(max_len=20000, max_pages=2000)
    n = size(b=b)
    assert n > 256
    assert attn(b=b, n=n - 1) == attn(b=b, ws=None) == kq.KQ_EWORKSPACE
    assert attn(b=b, ws=FAKE + 64, n=n) == kq.KQ_EALIGN


class _Cache(C.Structure):
    """kq::kv::Cache (kernels_amd/csrc/kq_internal.h)."""
    _fields_ = [(n, C.c_void_p) for n in ("k", "v", "k_exp", "v_exp")] + [(n, C.c_uint32) for n in ("n_pages", "heads", "page_log2", "block_log2")]


def test_workspace_covers_every_window():
    """What a call writes (libkq's own plan, declared in kq_internal.h) is within what kq_kv_attn_workspace_size said,
    whatever the window: over sizes where the launch takes its different forms, the largest among them."""
    need = kq.lib()["_ZN2kq15kv_attn_ws_needERKNS_2kv5CacheERKNS0_5BatchEjjj"]
    need.restype = C.c_size_t
    rng = np.random.default_rng(0)
    some = 0
    for _ in range(3000):
        heads, group = int(rng.choice([1, 2, 3, 8, 16, 64])), int(rng.choice([1, 2, 5, 8, 16, 64]))
        dim, page = int(rng.choice([64, 96, 128, 192, 256])), int(rng.choice([16, 64, 1024]))
        max_len, n_seq = int(2 ** rng.uniform(0, 31) * 0.99), int(2 ** rng.uniform(0, 14))
        max_q = int(2 ** rng.uniform(0, rng.choice([3, 12])))
        if n_seq * max_q * heads * group >= 2**31 - 2**16:
            continue
        b = batch_c(n_seq=n_seq, max_q=max_q, n_rows=n_seq * max_q, max_len=max(max_len, 1), max_pages=1 << 20)
        said = size(cache_c(heads=heads, head_dim=dim, page=page), b, heads * group)
        assert said > 0
        c = _Cache(FAKE, FAKE, FAKE, FAKE, 64, heads, page.bit_length() - 1, 4)
        for window in [0] + [int(2 ** rng.uniform(0, 31)) for _ in range(6)]:
            n = need(C.byref(c), C.byref(b), C.c_uint32(dim), C.c_uint32(group), C.c_uint32(window))
            assert n <= said, (heads, group, dim, max_len, n_seq, max_q, window)
            some += window > 0 and n > 0
    assert some > 1000


def test_workspace_size_refuses_what_the_call_refuses():
    for kw, _ in BAD_CACHE:
        assert size(cache_c(**kw)) == 0
    for kw, _ in BAD_BATCH:
        assert size(b=batch_c(**kw)) == 0
    assert size(q_heads=0) == size(q_heads=12) == size(q_heads=8 * 65) == 0
    assert size() >= 256


def test_launches_too_large():
    b = batch_c(n_seq=65535, max_q=0x7FFEFFFF, n_rows=0x7FFEFFFF)
    assert write(cache_c(heads=1024), b, rows_c(), rows_c()) == kq.KQ_EUNSUPPORTED
    assert write(cache_c(heads=1024), b, rows_c(row=1 << 17), rows_c(row=1 << 17), read=True) == kq.KQ_EUNSUPPORTED
    assert attn(b=b, n=(1 << 63)) == kq.KQ_EUNSUPPORTED


@pytest.mark.parametrize("n_seq,max_q,heads,group,dim,groups", [
    # rows of work, by the tiles of 16 or 32 rows of each (up to 64 rows) ...
    (16384, 1, 1024, 1, 64, 1 << 24), (65535, 1, 256, 64, 192, 65535 * 256 * 4), (32768, 2, 512, 16, 256, 2 << 24),
    # ... or by the 128s of rows
    (4096, 65, 1024, 2, 128, 2 << 22), (12000, 129, 1024, 1, 128, 12000 * 1024 * 2), (12000, 129, 1024, 1, 64, 12000 * 1024 * 2),
    (1 << 12, 250000, 1, 1, 96, 977 * 2 << 12)])
def test_launch_limits_of_the_attention(n_seq, max_q, heads, group, dim, groups):
    """2^24 workgroups of 256 threads, which HIP can't launch, are refused; a sixteenth of them is not."""
    q = rows_c(row=heads * group * dim, head=dim)
    for part in (1, 16):
        assert n_seq * max_q * heads * group // part < 2**31 - 2**16
        refused = groups // part >= 1 << 24
        b = batch_c(n_seq=n_seq // part, max_q=max_q, n_rows=0)
        c, d = cache_c(heads=heads, head_dim=dim), attn_c(q_heads=heads * group)
        assert (size(c, b, heads * group) == 0) == refused
        assert attn(c, b, d, q, q, n=1 << 62) == (kq.KQ_EUNSUPPORTED if refused else kq.KQ_OK)


@pytest.mark.parametrize("read,block", [(False, 16), (False, 256), (True, 256)])
def test_launch_limits_of_writing_and_reading(read, block):
    unit = 16 if read else block
    most = ((1 << 24) - 1) // 2 - 2  # blocks of 2 workgroups each: four heads' K and V
    for blocks, status in ((most, kq.KQ_OK), (most + 1, kq.KQ_EUNSUPPORTED)):
        b = batch_c(n_seq=1, max_q=min(blocks * unit, 2**31 - 2**17), n_rows=0)
        if b.max_q == blocks * unit:
            assert write(cache_c(heads=4, page=256, block=block), b, read=read) == status


def test_scale_whose_log2_is_no_number():
    assert attn(d=attn_c(scale=3e38)) == attn(d=attn_c(scale=-3e38)) == kq.KQ_EINVAL


def test_packed_structs():
    """What kq.py passes as bytes is what the C structs hold."""
    assert bytes(batch_c(pages=1, kv_len=2, q_start=3)) == kq._pack_batch(1, 2, 3, 2, 8, 3, 6, 100)
    assert bytes(rows_c(p=5, row=-3, head=2**40)) == kq._pack_rows(5, -3, 2**40)
    assert bytes(attn_c(sinks=9, scale=-0.5, window=7)) == kq._pack_attn(32, -0.5, True, 7, 9)


def test_python_tensors():
    c = kq.kv_cache(4, 2, 64, page=32, block=16, device="cpu")
    assert (c.page, c.block, c.heads, c.head_dim) == (32, 16, 2, 64)
    e = kq.kv_cache(4, 2, 96, dtype=torch.float8_e4m3fn, device="cpu")
    assert e._c.type == kq.KV_E4M3
    with pytest.raises(ValueError):
        kq.KVCache(c.k.float(), c.v, c.k_exp, c.v_exp)
    with pytest.raises(ValueError):
        kq.KVCache(c.k, c.v.transpose(3, 4), c.k_exp, c.v_exp)
    with pytest.raises(ValueError):
        kq.KVCache(c.k, c.v, c.k_exp[:, :, :1], c.v_exp)
    with pytest.raises(ValueError):
        kq.KVCache(c.k, c.v, c.k_exp.int(), c.v_exp)
    with pytest.raises(ValueError):
        kq.kv_cache(4, 2, 64, page=16, block=32, device="cpu")
    pages, n = torch.zeros((2, 4), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    kq.KVBatch(pages, n, 10)
    for bad in ((pages.long(), n), (pages.t(), n), (pages, n.long()), (pages[:1], n)):
        with pytest.raises(ValueError):
            kq.KVBatch(*bad, 10)
    with pytest.raises(ValueError):
        kq.KVBatch(pages, n, 10, q_start=n)
    with pytest.raises(ValueError):
        kq.KVBatch(pages, n, -1)
    b = kq.KVBatch(pages, n, 10)
    for shape in ((3, 2, 32), (3, 1, 64), (4, 2, 64), (3, 64), (3, 2, 64, 1)):
        with pytest.raises(ValueError):
            kq._kv_rows(torch.zeros(shape), (3, 2, 64), torch.float32, "k")
    with pytest.raises(ValueError):
        kq._kv_rows(torch.zeros((3, 2, 64)), (3, 2, 64), torch.float16, "k")
    with pytest.raises(ValueError):
        kq._kv_rows(torch.zeros((3, 64, 2)).transpose(1, 2), (3, 2, 64), torch.float32, "k")
    with pytest.raises(kq.KQError):
        kq.kv_attn_workspace_size(c, b, 3)


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
def test_oracle_codes(kind):
    """The oracle's rounding, against torch's conversions on the CPU and halfway values."""
    codes = np.arange(256, dtype=np.uint8)
    values = _kv.decode(codes, kind)
    fine = np.isfinite(values) & (values != 0) & (np.abs(values) <= _kv.LARGEST[kind])
    assert np.array_equal(_kv.encode(values[fine], kind), codes[fine])
    rng = np.random.default_rng(0)
    y = np.concatenate([rng.normal(0, 0.3 * _kv.LARGEST[kind], 5000), rng.normal(0, 0.01, 5000), (np.sort(values[fine])[1:] + np.sort(values[fine])[:-1]) / 2])
    y = y.astype(np.float32)
    t = torch.from_numpy(y).clamp(-_kv.LARGEST[kind], _kv.LARGEST[kind])
    want = t.round().to(torch.int8).view(torch.uint8) if kind == "i8" else t.to(torch.float8_e4m3fn).view(torch.uint8)
    assert np.array_equal(_kv.decode(_kv.encode(y.astype(np.float64), kind), kind), _kv.decode(want.numpy(), kind))


def test_oracle_exponents():
    for kind in ("i8", "e4m3"):
        big = _kv.LARGEST[kind]
        assert _kv.exponent(0.0, kind) == -64
        assert _kv.exponent(big, kind) == 0 and _kv.exponent(np.nextafter(big, 1e9), kind) == 1
        assert _kv.exponent(big / 2, kind) == -1
        assert _kv.exponent(3.3e38, kind) == _kv.MAX_EXP[kind]


@pytest.mark.parametrize("rows,heads,row,head,overlap", [
    (6, 32, 128, 128, True), (2, 2, 128, 128, True), (6, 32, 31 * 128, 128, True), (6, 32, 32 * 128 - 8, 128, True),
    (6, 32, 128, 5 * 128, True), (6, 32, 128, 6 * 128 - 8, True), (3, 4, 3 * 128, 2 * 128, True), (4, 3, 2 * 128, 3 * 128, True),
    (2**20, 2, 128, 2**20 * 128 - 8, True), (65535, 32, 8 * 1001, 8 * 1003, True), (2, 32, 2**62, 2**61, True),
    (6, 32, 32 * 128, 128, False), (6, 32, 128, 6 * 128, False), (6, 32, 40 * 128, 128, False), (2, 2, 3 * 128, 2 * 128, False),
    (1, 32, 0, 128, False), (2, 32, 2**62, 2**40, False), (2**20, 2, 128, 2**20 * 128, False), (6, 1, 128, 0, False)])
def test_rows_and_heads_that_meet(rows, heads, row, head, overlap):
    """Outputs whose rows and heads share elements are refused, whichever of the strides is the larger; those that lie
    between one another without sharing any are not."""
    # by search, where there are few enough
    if rows * heads <= 4096 and max(row, head) < 2**40:
        at = np.sort((np.arange(rows)[:, None] * row + np.arange(heads) * head).reshape(-1))
        assert (np.diff(at).min() < 128) == overlap
    b, r = batch_c(n_seq=1, max_q=1, n_rows=rows), rows_c(row=row, head=head)
    q = rows_c(row=0, head=0)
    assert attn(cache_c(heads=1), b, attn_c(q_heads=heads), q, r, ws=None) == (kq.KQ_EINVAL if overlap else kq.KQ_EWORKSPACE)
    if overlap:
        c, fine = cache_c(heads=heads), rows_c(row=2**30, head=128)
        assert write(c, b, r, fine, read=True) == write(c, b, fine, r, read=True) == kq.KQ_EINVAL


@pytest.mark.parametrize("starts", [False, True])
def test_python_workspace_size_of_bounds_too_large(starts):
    """n_seq * max_q beyond 32 bits: refused like any bounds that no launch can have."""
    n = 65535
    c, length = kq.kv_cache(4, 1, 64, device="cpu"), torch.zeros(n, dtype=torch.int32)
    b = kq.KVBatch(torch.zeros((n, 1), dtype=torch.int32), length, 16, max_q=1 << 17,
                   q_start=torch.zeros(n + 1, dtype=torch.int32) if starts else None)
    with pytest.raises(kq.KQError):
        kq.kv_attn_workspace_size(c, b, 1)


@pytest.mark.parametrize("read,block", [(False, 16), (False, 64), (False, 256), (True, 16), (True, 256)])
def test_launch_limits_of_many_heads(read, block):
    """Blocks of 512 workgroups each (1024 heads' K and V): few enough tokens for blocks of 256 too."""
    unit = 16 if read else block
    most = ((1 << 24) - 1) // 512 - 2
    for blocks, status in ((most, kq.KQ_OK), (most + 1, kq.KQ_EUNSUPPORTED)):
        b = batch_c(n_seq=1, max_q=blocks * unit, n_rows=0)
        assert b.max_q < 0x7FFF0000
        assert write(cache_c(heads=1024, page=256, block=block), b, read=read) == status


def test_launch_limits_as_documented():
    """kq_kv_attn_workspace_size refuses what include/kq.h says, over random bounds beside the limits."""
    rng = np.random.default_rng(1)
    seen = set()
    for _ in range(20000):
        n_seq, heads, group = int(2 ** rng.uniform(0, 16)) - 1 or 1, int(2 ** rng.uniform(0, 10)), int(rng.choice([1, 3, 8, 40, 64]))
        dim, max_q = int(rng.choice([64, 96, 128, 192, 256])), int(2 ** rng.uniform(0, rng.choice([2, 8, 20])))
        rows = max_q * group
        if rows <= 64:
            each = 16 if rows <= 16 or dim in (192, 256) else 32
            groups = -(-n_seq * heads // 8) * 8 * -(-rows // each)
        elif dim in (96, 128) and rows > 128:
            groups = n_seq * heads * -(-rows // 256) * 2
        else:
            groups = n_seq * heads * -(-rows // 128)
        refused = groups >= 1 << 24 or n_seq * max_q * heads * group >= 2**31 - 2**16
        b = batch_c(n_seq=n_seq, max_q=max_q, n_rows=0)
        assert (size(cache_c(heads=heads, head_dim=dim), b, heads * group) == 0) == refused, (n_seq, heads, group, dim, max_q)
        seen.add((refused, rows <= 64))
    assert len(seen) == 4
