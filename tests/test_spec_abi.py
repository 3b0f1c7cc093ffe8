"""The calls of a speculative step on the CPU: what the host refuses before any launch, and
what it computes itself."""
import ctypes as C

import numpy as np
import pytest

from kernels_amd import kq
from tests.test_kv_abi import _Cache, BAD_BATCH, BAD_BATCH_P, BAD_CACHE, BAD_CACHE_P, FAKE, attn_c, batch_c, cache_c, rows_c


def rope_c(**kw):
    a = dict(inv_freq=FAKE, rot=128, layout=0, amplitude=1.0, inverse=0)
    a.update(kw)
    return kq._RopeC(**a)


def rope(d=None, pos=FAKE, X=None, Y=None, n=6, heads=8, dim=128, dt=kq.F16):
    return kq.lib().kq_rope(C.byref(d or rope_c()), pos, C.byref(X or rows_c()), C.byref(Y or rows_c(p=FAKE * 2)), n, heads, dim, dt, None)


def write(c=None, b=None, d=None, pos=None, Q=None, Qo=None, q_heads=32, K=None, V=None, dt=kq.F16, q=True):
    Q, Qo = Q or rows_c(row=4096), Qo or rows_c(p=FAKE * 2, row=4096)
    return kq.lib().kq_kv_write_rope(C.byref(c or cache_c()), C.byref(b or batch_c()), C.byref(d or rope_c()), pos,
                                     C.byref(Q) if q else None, C.byref(Qo) if q else None, q_heads, C.byref(K or rows_c()),
                                     C.byref(V or rows_c()), dt, None)


@pytest.mark.parametrize("kw,status", [
    (dict(inv_freq=None), kq.KQ_ENULL), (dict(inv_freq=FAKE + 2), kq.KQ_EALIGN), (dict(rot=0), kq.KQ_EINVAL), (dict(rot=63), kq.KQ_EINVAL),
    (dict(rot=130), kq.KQ_EINVAL), (dict(layout=2), kq.KQ_EINVAL), (dict(amplitude=float("nan")), kq.KQ_EINVAL),
    (dict(amplitude=float("inf")), kq.KQ_EINVAL)])
def test_bad_rope(kw, status):
    assert rope(rope_c(**kw)) == write(d=rope_c(**kw)) == status


@pytest.mark.parametrize("kw,status", [
    (dict(dim=0), kq.KQ_EINVAL), (dict(dim=132), kq.KQ_EINVAL), (dict(dim=520), kq.KQ_EUNSUPPORTED), (dict(heads=0), kq.KQ_EINVAL),
    (dict(heads=65536), kq.KQ_EINVAL), (dict(n=0x7FFF0000), kq.KQ_EINVAL), (dict(dt=3), kq.KQ_EUNSUPPORTED), (dict(pos=None), kq.KQ_ENULL),
    (dict(pos=FAKE + 2), kq.KQ_EALIGN), (dict(X=rows_c(p=None)), kq.KQ_ENULL), (dict(Y=rows_c(p=FAKE + 8)), kq.KQ_EALIGN),
    (dict(X=rows_c(row=1028)), kq.KQ_EINVAL), (dict(Y=rows_c(row=0)), kq.KQ_EINVAL), (dict(Y=rows_c(head=64)), kq.KQ_EINVAL),
    (dict(X=rows_c(row=2048), Y=rows_c(row=1024)), kq.KQ_EINVAL), (dict(X=rows_c(head=256, row=2048), Y=rows_c(row=2048)), kq.KQ_EINVAL)])
def test_bad_rows(kw, status):
    assert rope(**kw) == status


def test_rope_of_no_rows_and_launch_limits():
    none = rows_c(p=None)
    assert rope(n=0, X=none, Y=none, pos=None) == kq.KQ_OK
    assert rope(n=0, X=none, Y=none, dt=7) == kq.KQ_EUNSUPPORTED
    assert rope(n=2**27, X=rows_c(row=1 << 17), Y=rows_c(p=FAKE * 2, row=1 << 17)) == kq.KQ_EUNSUPPORTED


def test_null_structs():
    L = kq.lib()
    r, d = rows_c(), rope_c()
    assert L.kq_rope(None, FAKE, C.byref(r), C.byref(r), 6, 8, 128, 0, None) == kq.KQ_ENULL
    assert L.kq_rope(C.byref(d), FAKE, None, C.byref(r), 6, 8, 128, 0, None) == kq.KQ_ENULL
    assert L.kq_kv_write_rope(C.byref(cache_c()), C.byref(batch_c()), None, None, None, None, 0, C.byref(r), C.byref(r), 0, None) == kq.KQ_ENULL
    assert L.kq_kv_write_rope(C.byref(cache_c()), C.byref(batch_c()), C.byref(d), None, C.byref(rows_c(row=4096)), None, 32, C.byref(r), C.byref(r), 0, None) == kq.KQ_ENULL


@pytest.mark.parametrize("kw,status", BAD_CACHE + BAD_CACHE_P)
def test_bad_cache(kw, status):
    assert write(cache_c(**kw)) == status


@pytest.mark.parametrize("kw,status", BAD_BATCH + BAD_BATCH_P)
def test_bad_batch(kw, status):
    assert write(b=batch_c(**kw)) == status


@pytest.mark.parametrize("kw,status", [
    (dict(d=rope_c(rot=24)), kq.KQ_EUNSUPPORTED), (dict(dt=kq.F32), kq.KQ_EUNSUPPORTED), (dict(pos=FAKE + 2), kq.KQ_EALIGN),
    (dict(q_heads=0), kq.KQ_EINVAL), (dict(q_heads=65536), kq.KQ_EINVAL), (dict(Q=rows_c(p=None)), kq.KQ_ENULL),
    (dict(Qo=rows_c(row=120)), kq.KQ_EINVAL), (dict(Qo=rows_c(p=FAKE + 8, row=4096)), kq.KQ_EALIGN), (dict(Q=rows_c(row=8192), Qo=rows_c(row=4096)), kq.KQ_EINVAL),
    (dict(K=rows_c(p=None)), kq.KQ_ENULL), (dict(V=rows_c(row=1028)), kq.KQ_EINVAL)])
def test_bad_write(kw, status):
    assert write(**kw) == status


def test_write_of_no_rows_and_launch_limits():
    none = rows_c(p=None)
    assert write(b=batch_c(n_rows=0), K=none, V=none, Q=none, Qo=none) == kq.KQ_OK
    assert write(b=batch_c(n_rows=0), K=none, V=none, q=False) == kq.KQ_OK
    # without queries the blocks fit; the queries' rows are too many
    b = batch_c(n_rows=0, max_q=2**24, max_len=2**24, max_pages=2**20)
    assert write(b=b, K=none, V=none, q=False) == kq.KQ_OK
    assert write(b=b, K=none, V=none, Q=none, Qo=none) == kq.KQ_EUNSUPPORTED


# ---- frequencies, which the host computes

def freqs(rot=64, **kw):
    f, a = kq.rope_freqs(rot, device="cpu", **kw)
    return f.double().numpy(), a


def test_freqs_plain_linear_ntk():
    i = np.arange(32)
    want = 10000.0 ** (-2 * i / 64)
    assert np.allclose(freqs()[0], want, rtol=2**-24, atol=0) and freqs()[1] == 1.0
    assert np.allclose(freqs(kind="linear", factor=4.0)[0], want / 4, rtol=2**-24, atol=0)
    got = freqs(kind="ntk", factor=8.0)[0]
    # the fastest pair as it is, the slowest slower by the factor
    assert got[0] == 1.0 and abs(got[-1] * 8.0 / want[-1] - 1) < 2**-22


def test_freqs_bands():
    want, got = freqs(base=500000.0)[0], freqs(base=500000.0, kind="bands", factor=8.0, low=1.0, high=4.0, original=8192.0)[0]
    turns = 8192.0 * want / (2 * np.pi)
    assert np.array_equal(got[turns > 4], want[turns > 4]) and (turns > 4).any()
    assert np.allclose(got[turns < 1], want[turns < 1] / 8, rtol=2**-22, atol=0) and (turns < 1).any()
    mid = (turns >= 1) & (turns <= 4)
    share = (turns[mid] - 1) / 3
    assert np.allclose(got[mid], want[mid] * share + want[mid] / 8 * (1 - share), rtol=2**-21, atol=0) and mid.any()


def test_freqs_yarn():
    want, (got, a) = freqs()[0], freqs(kind="yarn", factor=16.0, original=4096.0)
    assert abs(a - (0.1 * np.log(16.0) + 1)) < 2**-50
    c = [64 * np.log(4096 / (n * 2 * np.pi)) / (2 * np.log(10000.0)) for n in (32.0, 1.0)]
    lo, hi = np.floor(c[0]), np.ceil(c[1])
    r = np.clip((np.arange(32) - lo) / (hi - lo), 0, 1)
    assert np.allclose(got, want * (1 - r) + want / 16 * r, rtol=2**-22, atol=0)
    assert got[0] == 1.0 and got[-1] < want[-1] / 15
    # a context so short that both ends meet
    f, _ = freqs(kind="yarn", factor=2.0, original=1.0)
    assert np.isfinite(f).all()


@pytest.mark.parametrize("kw", [dict(rot=0), dict(rot=3), dict(rot=514), dict(base=1.0), dict(base=float("nan")), dict(base=float("inf")),
                                dict(kind="linear", factor=0.5), dict(kind="linear", factor=float("nan")), dict(kind="ntk", rot=2, factor=2.0),
                                dict(kind="bands", factor=2.0), dict(kind="bands", factor=2.0, original=100.0, low=4.0, high=4.0),
                                dict(kind="yarn", factor=2.0, original=float("inf")), dict(kind="yarn", factor=2.0, original=-1.0)])
def test_freqs_refused(kw):
    with pytest.raises(kq.KQError) as e:
        freqs(**kw)
    assert e.value.status == kq.KQ_EINVAL


def test_freqs_nulls_and_kinds():
    L, d, a = kq.lib(), kq._RopeScalingC(0, 64, 1e4, 1, 1, 4, 0), C.c_double()
    out = (C.c_float * 32)()
    assert L.kq_rope_freqs(None, out, C.byref(a)) == L.kq_rope_freqs(C.byref(d), None, C.byref(a)) == L.kq_rope_freqs(C.byref(d), out, None) == kq.KQ_ENULL
    d.kind = 5
    assert L.kq_rope_freqs(C.byref(d), out, C.byref(a)) == kq.KQ_EINVAL
    with pytest.raises(ValueError):
        kq.rope_freqs(64, kind="other", device="cpu")


# ---- trees

def nodes_c(**kw):
    a = dict(mask=FAKE, pos=FAKE, words=1)
    a.update(kw)
    return kq._KVNodesC(**a)


def tree(b=None, parent=FAKE, mask=FAKE, words=1, pos=None, window=0):
    return kq.lib().kq_kv_tree(C.byref(b or batch_c()), parent, mask, words, pos, window, None)


def attn(c=None, b=None, d=None, t=None, Q=None, O=None, dt=kq.F16, lse=None, ws=FAKE, n=1 << 30):
    return kq.lib().kq_kv_attn_tree(C.byref(c or cache_c()), C.byref(b or batch_c()), C.byref(d or attn_c()), C.byref(t or nodes_c()),
                                    C.byref(Q or rows_c(row=4096)), C.byref(O or rows_c(row=4096)), dt, lse, ws, n, None)


@pytest.mark.parametrize("kw,status", BAD_BATCH + [(dict(kv_len=None), kq.KQ_ENULL), (dict(kv_len=FAKE + 1), kq.KQ_EALIGN), (dict(q_start=FAKE + 2), kq.KQ_EALIGN),
                                                   (dict(max_q=1025), kq.KQ_EUNSUPPORTED)])
def test_tree_bad_batch(kw, status):
    assert tree(batch_c(**kw), words=64) == status


@pytest.mark.parametrize("kw,status", [
    (dict(parent=None), kq.KQ_ENULL), (dict(mask=None), kq.KQ_ENULL), (dict(parent=FAKE + 2), kq.KQ_EALIGN), (dict(mask=FAKE + 1), kq.KQ_EALIGN),
    (dict(pos=FAKE + 2), kq.KQ_EALIGN), (dict(words=0), kq.KQ_EINVAL), (dict(words=2**31), kq.KQ_EINVAL), (dict(b=batch_c(max_q=33)), kq.KQ_EINVAL)])
def test_bad_tree(kw, status):
    assert tree(**kw) == status


@pytest.mark.parametrize("kw,status", BAD_CACHE + BAD_CACHE_P)
def test_attention_bad_cache(kw, status):
    assert attn(cache_c(**kw)) == status


@pytest.mark.parametrize("kw,status", BAD_BATCH + BAD_BATCH_P)
def test_attention_bad_batch(kw, status):
    assert attn(b=batch_c(**kw), t=nodes_c(words=1 << 20)) in (status, kq.KQ_EUNSUPPORTED if kw.get("max_q", 0) > 1024 else status)


@pytest.mark.parametrize("kw,status", [
    (dict(t=nodes_c(mask=None)), kq.KQ_ENULL), (dict(t=nodes_c(pos=None), d=attn_c(window=5)), kq.KQ_ENULL), (dict(t=nodes_c(mask=FAKE + 2)), kq.KQ_EALIGN),
    (dict(t=nodes_c(pos=FAKE + 2)), kq.KQ_EALIGN), (dict(t=nodes_c(words=0)), kq.KQ_EINVAL), (dict(b=batch_c(max_q=1025), t=nodes_c(words=64)), kq.KQ_EUNSUPPORTED),
    (dict(dt=kq.F32), kq.KQ_EUNSUPPORTED), (dict(d=attn_c(q_heads=12)), kq.KQ_EINVAL), (dict(d=attn_c(scale=float("nan"))), kq.KQ_EINVAL),
    (dict(ws=None), kq.KQ_EWORKSPACE), (dict(n=0), kq.KQ_EWORKSPACE), (dict(ws=FAKE + 16), kq.KQ_EALIGN), (dict(lse=FAKE + 2), kq.KQ_EALIGN),
    (dict(O=rows_c(row=0)), kq.KQ_EINVAL)])
def test_bad_attention(kw, status):
    assert attn(**kw) == status


def test_tree_of_no_rows():
    none = rows_c(p=None)
    assert tree(batch_c(n_rows=0), parent=None, mask=None) == kq.KQ_OK
    assert attn(b=batch_c(n_rows=0), t=nodes_c(mask=None, pos=None), Q=none, O=none, d=attn_c(causal=0, window=3)) == kq.KQ_OK
    L = kq.lib()
    assert L.kq_kv_tree(None, FAKE, FAKE, 1, None, 0, None) == kq.KQ_ENULL
    r = rows_c(row=4096)
    assert L.kq_kv_attn_tree(C.byref(cache_c()), C.byref(batch_c()), C.byref(attn_c()), None, C.byref(r), C.byref(r), 0, None, FAKE, 1 << 30, None) == kq.KQ_ENULL


def size(c=None, b=None, q_heads=32):
    return kq.lib().kq_kv_attn_tree_workspace_size(C.byref(c or cache_c()), C.byref(b or batch_c()), q_heads)


def test_tree_workspace():
    for kw, _ in BAD_CACHE:
        assert size(cache_c(**kw)) == 0
    for kw, _ in BAD_BATCH + [(dict(max_q=1025), 0)]:
        assert size(b=batch_c(**kw)) == 0
    assert size(q_heads=0) == size(q_heads=12) == size(q_heads=8 * 65) == 0
    b = batch_c(n_seq=1, max_q=64, max_len=9000, n_rows=64)
    n = size(b=b)
    assert n > 256 and n % 256 == 0
    assert attn(b=b, t=nodes_c(words=2), n=n - 1) == kq.KQ_EWORKSPACE


def test_tree_workspace_covers_every_window():
    """What a call writes is within what kq_kv_attn_tree_workspace_size said, over the launch's forms."""
    need = kq.lib()["_ZN2kq15kv_tree_ws_needERKNS_2kv5CacheERKNS0_5BatchEjjj"]
    need.restype = C.c_size_t
    rng = np.random.default_rng(0)
    some = 0
    for _ in range(3000):
        heads, group = int(rng.choice([1, 2, 3, 8, 16, 64])), int(rng.choice([1, 2, 5, 8, 16, 64]))
        dim, page = int(rng.choice([64, 96, 128, 192, 256])), int(rng.choice([16, 64, 1024]))
        max_len, n_seq = int(2 ** rng.uniform(0, 31) * 0.99), int(2 ** rng.uniform(0, 14))
        max_q = int(2 ** rng.uniform(0, rng.choice([3, 10])))
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


# ---- verification, and the kept rows

def draft(**kw):
    a = dict(p=FAKE, q=FAKE, p_row=100, q_row=100, q_index=FAKE, token=FAKE, parent=FAKE, start=FAKE, u=FAKE, n_seq=2, max_q=3, n_rows=6,
             n_q=6, vocab=100)
    a.update(kw)
    return kq._pack_draft(*((v or 0) for v in a.values()))


def verify(d=None, keep=FAKE, n_keep=FAKE, out=FAKE, ws=FAKE, n=1 << 40):
    return kq.lib().kq_draft_verify(d or draft(), keep, n_keep, out, ws, n, None)


@pytest.mark.parametrize("kw,status", [
    (dict(n_seq=0), kq.KQ_EINVAL), (dict(n_seq=65536), kq.KQ_EINVAL), (dict(max_q=0), kq.KQ_EINVAL), (dict(max_q=1025), kq.KQ_EUNSUPPORTED),
    (dict(vocab=0), kq.KQ_EINVAL), (dict(vocab=0x7FFF0000), kq.KQ_EUNSUPPORTED), (dict(n_rows=0x7FFF0000), kq.KQ_EINVAL),
    (dict(start=None, n_rows=5), kq.KQ_EINVAL), (dict(p=None), kq.KQ_ENULL), (dict(token=None), kq.KQ_ENULL), (dict(u=None), kq.KQ_ENULL),
    (dict(p_row=-1), kq.KQ_EINVAL), (dict(q_row=-100), kq.KQ_EINVAL), (dict(q_index=None, n_q=5), kq.KQ_EINVAL), (dict(n_q=0x7FFF0000), kq.KQ_EINVAL),
    (dict(p=FAKE + 2), kq.KQ_EALIGN), (dict(q=FAKE + 1), kq.KQ_EALIGN), (dict(q_index=FAKE + 2), kq.KQ_EALIGN), (dict(token=FAKE + 2), kq.KQ_EALIGN),
    (dict(parent=FAKE + 2), kq.KQ_EALIGN), (dict(start=FAKE + 2), kq.KQ_EALIGN), (dict(u=FAKE + 2), kq.KQ_EALIGN)])
def test_bad_draft(kw, status):
    assert verify(draft(**kw)) == status


@pytest.mark.parametrize("kw,status", [
    (dict(keep=None), kq.KQ_ENULL), (dict(n_keep=None), kq.KQ_ENULL), (dict(out=None), kq.KQ_ENULL), (dict(keep=FAKE + 2), kq.KQ_EALIGN),
    (dict(n_keep=FAKE + 2), kq.KQ_EALIGN), (dict(out=FAKE + 1), kq.KQ_EALIGN), (dict(ws=None), kq.KQ_EWORKSPACE), (dict(n=255), kq.KQ_EWORKSPACE),
    (dict(ws=FAKE + 16), kq.KQ_EALIGN)])
def test_bad_verify(kw, status):
    assert verify(**kw) == status


def test_verify_workspace():
    size = kq.lib().kq_draft_verify_workspace_size
    assert size(0, 3, 100) == size(65536, 3, 100) == size(2, 0, 100) == size(2, 1025, 100) == size(2, 3, 0) == size(2, 3, 0x7FFF0000) == 0
    assert kq.lib().kq_draft_verify(None, FAKE, FAKE, FAKE, FAKE, 1 << 40, None) == kq.KQ_ENULL
    for n_seq, max_q, vocab in ((1, 1, 1), (2, 3, 100), (65535, 1024, 300000), (1, 1024, 0x7FFEFFFF)):
        n = size(n_seq, max_q, vocab)
        assert n % 256 == 0 and n >= n_seq * (16 * max_q + 8 * -(-vocab // 4096) + 16)
    d = draft(n_seq=64, max_q=5, n_rows=320, vocab=128256, n_q=320)
    assert verify(d, n=size(64, 5, 128256) - 1) == kq.KQ_EWORKSPACE


def keep(c=None, b=None, rows=FAKE, n=FAKE):
    return kq.lib().kq_kv_keep(C.byref(c or cache_c()), C.byref(b or batch_c()), rows, n, None)


@pytest.mark.parametrize("kw,status", BAD_CACHE + BAD_CACHE_P)
def test_keep_bad_cache(kw, status):
    assert keep(cache_c(**kw)) == status


@pytest.mark.parametrize("kw,status", BAD_BATCH + BAD_BATCH_P + [(dict(max_q=1025), kq.KQ_EUNSUPPORTED)])
def test_keep_bad_batch(kw, status):
    assert keep(b=batch_c(**kw)) == status


@pytest.mark.parametrize("kw,status", [(dict(rows=None), kq.KQ_ENULL), (dict(n=None), kq.KQ_ENULL), (dict(rows=FAKE + 2), kq.KQ_EALIGN),
                                       (dict(n=FAKE + 2), kq.KQ_EALIGN), (dict(b=batch_c(n_rows=0)), kq.KQ_OK)])
def test_bad_keep(kw, status):
    assert keep(**kw) == status


# ---- the Python layer's own refusals (on the CPU: every tensor is on device -1)

@pytest.fixture
def no_gpu(monkeypatch):
    """The wrappers' checks without a device: calls that pass them raise KeyError in place of a launch."""
    import torch

    class Lib:
        def __getattr__(self, name):
            raise KeyError(name)

    monkeypatch.setattr(kq, "_stream", lambda s: 0)
    monkeypatch.setattr(kq, "_current", (lambda d: 0, lambda: -1))
    monkeypatch.setattr(kq, "_lib", Lib())
    return torch


def test_python_refusals(no_gpu):
    t = no_gpu
    i32, f32, f16 = t.int32, t.float32, t.float16
    z = lambda *s, dtype=i32: t.zeros(s, dtype=dtype)  # noqa: E731
    good = dict(p=z(6, 50, dtype=f32), token=z(6), u=z(6, dtype=f32), keep=z(2, 3), n_keep=z(2), out=z(2, 3), ws=0, ws_bytes=0)
    with pytest.raises(KeyError):
        kq.draft_verify(**good)
    with pytest.raises(KeyError):
        kq.draft_verify(**good, q=z(9, 50, dtype=f32), q_index=z(6), parent=z(6), start=z(3))
    for kw in (dict(p=z(6, 50)), dict(p=z(6, dtype=f32)), dict(p=z(50, 6, dtype=f32).t()), dict(token=z(5)), dict(token=z(6, dtype=t.int64)),
               dict(u=z(6)), dict(u=z(7, dtype=f32)), dict(keep=z(2, 4)), dict(keep=z(3, 2).t()), dict(n_keep=z(3)), dict(out=z(2, 3, dtype=t.int64)),
               dict(parent=z(5)), dict(start=z(2)), dict(q=z(5, 50, dtype=f32)), dict(q=z(6, 49, dtype=f32)), dict(q_index=z(7)),
               dict(q=z(6, 50, dtype=f16))):
        with pytest.raises(ValueError):
            kq.draft_verify(**{**good, **kw})
    x, pos, f = z(4, 2, 64, dtype=f16), z(4), kq.Rope(z(32, dtype=f32))
    with pytest.raises(KeyError):
        kq.rope(x, x, pos, f)
    for a in ((z(4, 64, dtype=f16), x, pos), (x, z(4, 2, 32, dtype=f16), pos), (x, z(4, 2, 64, dtype=f32), pos), (x, x, z(3)), (x, x, z(4, dtype=t.int64)),
              (x, x, z(8)[::2]), (x.transpose(1, 2), x.transpose(1, 2), pos)):
        with pytest.raises(ValueError):
            kq.rope(*a, f)
    for a in (z(32), z(2, 32, dtype=f32)):
        with pytest.raises(ValueError):
            kq.Rope(a)
    cache = kq.KVCache(z(4, 2, 16, 64, dtype=t.int8), z(4, 2, 1, 64, 16, dtype=t.int8), *(z(4, 2, 1, dtype=t.uint8) for _ in "kv"))
    b = kq.KVBatch(z(2, 2), z(2), 32, max_q=2)
    k, q = x, z(4, 6, 64, dtype=f16)
    with pytest.raises(KeyError):
        kq.kv_write_rope(cache, b, f, k, k, q=q, q_out=q, pos=pos)
    for kw in (dict(q=q), dict(q_out=q), dict(q=z(3, 6, 64, dtype=f16), q_out=q), dict(q=q, q_out=z(4, 5, 64, dtype=f16)),
               dict(q=q.bfloat16(), q_out=q.bfloat16()), dict(pos=z(3))):
        with pytest.raises(ValueError):
            kq.kv_write_rope(cache, b, f, k, k, **kw)
    with pytest.raises(ValueError):
        kq.kv_write_rope(cache, b, f, z(4, 3, 64, dtype=f16), k)
    with pytest.raises(KeyError):
        kq.kv_keep(cache, b, z(2, 2), z(2))
    for a in ((z(2, 3), z(2)), (z(2, 2), z(3)), (z(2, 2, dtype=t.int64), z(2))):
        with pytest.raises(ValueError):
            kq.kv_keep(cache, b, *a)
    tree = kq.KVTree(z(4, 1), z(4))
    with pytest.raises(KeyError):
        kq.kv_attn_tree(cache, b, tree, q, q.clone(), 0, 0)
    for bad in (kq.KVTree(z(3, 1)),):
        with pytest.raises(ValueError):
            kq.kv_attn_tree(cache, b, bad, q, q.clone(), 0, 0)
    for a in ((z(4), None), (z(4, 1, dtype=t.int64), None), (z(4, 1), z(3))):
        with pytest.raises(ValueError):
            kq.KVTree(*a)
    for kw in (dict(parent=z(3)), dict(window=-1), dict(pos=z(3)), dict(mask=z(4))):
        with pytest.raises(ValueError):
            kq.kv_tree(b, **{**dict(parent=z(4), mask=z(4, 1)), **kw})


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
def test_tree_workspace_at_most(dim):
    """The sizes that kq.h names: some 70 MB while a sequence and head has up to 32768 rows, and some 140 beyond."""
    most = {False: 0, True: 0}
    for heads in (1, 2, 8, 64):
        for group in (1, 3, 8, 33, 64):
            for max_q in (1, 2, 9, 33, 128, 257, 512, 513, 516, 1000, 1024):
                for n_seq in (1, 7, 200):
                    for max_len in (100, 3000, 2**20):
                        b = batch_c(n_seq=n_seq, max_q=max_q, n_rows=n_seq * max_q, max_len=max_len, max_pages=2**17)
                        many = max_q * group > 32768
                        most[many] = max(most[many], size(cache_c(head_dim=dim, heads=heads), b, heads * group))
    assert 0 < most[False] <= 70e6 and most[True] <= 140e6
    assert dim < 192 or most[True] > 100e6


def test_freqs_refused_without_memory():
    """A rot that is refused takes no memory for its frequencies first."""
    import tracemalloc
    tracemalloc.start()
    try:
        for rot in (514, 2**20, 2**26):
            with pytest.raises(kq.KQError):
                kq.rope_freqs(rot, device="cpu")
        assert tracemalloc.get_traced_memory()[1] < 2**20
    finally:
        tracemalloc.stop()
    got, _ = kq.rope_freqs(512, device="cpu")
    assert got.shape == (256,)
