"""The key/value cache's exponent bytes from 0 to 255, as a cache from elsewhere may
hold them: a code c of a block stands for c * 2^(byte - 127) whatever the byte,
against the 64-bit oracle (tests/_kv.py)."""
import numpy as np
import pytest
import torch

from kernels_amd import kq
from tests import _kv
from tests.test_gpu_kv import DTYPES, EPS, Batch, same_cache, to, upload

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 96])
def test_read(gpu, dim, kind, out):
    """A block of every byte. The values are float32 numbers (the smallest 2^-136) or beyond its largest, which a
    type's largest then stands for: float64 -> float32 loses nothing, and one rounding is left."""
    rng = np.random.default_rng(dim)
    seqs = [(4096, 4096), (100, 30)]
    b = Batch(gpu, seqs, 16, rng)
    oracle = _kv.Cache(b.n_pages, 1, dim, kind=kind)
    oracle.fill(rng)
    for w in "kv":
        oracle.codes[w][..., ::7] = 0
        oracle.exps[w][b.table[0], 0, 0] = rng.permutation(256)
    cache = upload(oracle, gpu)
    got = {w: torch.full((b.rows, 1, dim), 7.0, dtype=DTYPES[out], device=gpu) for w in "kv"}
    kq.kv_read(cache, b.c, got["k"], got["v"])
    torch.cuda.synchronize()
    top = torch.finfo(DTYPES[out]).max
    for w in "kv":
        for i, (n, m) in enumerate(seqs):
            want = torch.from_numpy(oracle.read(w, b.table[i], n, m)).clamp(-top, top).float().to(DTYPES[out])
            have = got[w][b.starts[i]:b.starts[i + 1]].cpu()
            bad = (have != want).nonzero()
            first = tuple(bad[0].tolist()) if len(bad) else None
            assert first is None, (w, i, first, have[first].item(), want[first].item(), len(bad))


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim,block", [(64, 16), (128, 32)])
def test_write(gpu, dim, block, dtype, kind):
    """Tokens appended to blocks of any byte: the byte stays where it is the larger, and the new codes are x / 2^(byte - 127)."""
    rng = np.random.default_rng(dim)
    was = (0, 1, 10, 62, 63, 64, 127, 190, 246, 248, 252, 253, 254, 255)
    seqs = [(block + 9, 4)] * len(was)
    b = Batch(gpu, seqs, block, rng)
    oracle = _kv.Cache(b.n_pages, 1, dim, block, block, kind)
    oracle.fill(rng)
    for i, e in enumerate(was):
        for w in "kv":
            oracle.exps[w][b.table[i, 1]] = e
    cache = upload(oracle, gpu)
    size = 3.3e38 if dtype == "bf16" else 6e4
    x = {w: to(np.sign(rng.normal(0, 1, (b.rows, 1, dim))) * size * 2.0 ** -rng.integers(0, 9, (b.rows, 1, dim)), dtype, gpu) for w in "kv"}
    kq.kv_write(cache, b.c, x["k"][0], x["v"][0])
    torch.cuda.synchronize()
    for w in "kv":
        for i, (n, m) in enumerate(seqs):
            oracle.write(w, x[w][1][b.starts[i]:b.starts[i + 1]], b.table[i], n, m)
    same_cache(cache, oracle)
