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
