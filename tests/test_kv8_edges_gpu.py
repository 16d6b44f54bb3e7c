"""Edges of the paged 8-bit KV cache: tiles of padding, value scales far apart,
queries that are not finite, limits of the calls. Helpers, bounds and the
oracle are test_kv8_gpu.py's."""
import numpy as np
import pytest
import torch

import lowbit_b200 as lb
import test_kv8_gpu as G
from lowbit_b200 import kernels as K
from oracle import kv8_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)
    K.device_status(reset=True)


@pytest.mark.parametrize("dt", G.TYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
def test_tiles_of_padding_are_zero(dt, d):
    """Prompts whose whole row tiles see nothing (before position 0, or past the table under a window): exact
    zeros every time, and the other rows are right."""
    rng = np.random.default_rng(40)
    b, new, page = 12, 150, 64
    pool = G.host_pool(rng, 5 * b, 4, page, d)
    cache, table = G.device_pool(pool), rng.permutation(5 * b).reshape(b, 5)
    pos = np.array([0, -150, 70, -1000, 33, -130, 7, -149, 100, -150, 150, -64])
    q = torch.randn((b * new, 8, d), device="cuda").to(G.TYPES[dt])
    at = (pos[:, None] + np.arange(new)).reshape(-1)
    ref, mag, size = R.attention(pool, q.double().cpu().numpy(), table, pos)
    out = torch.empty_like(q)
    for _ in range(20):
        out.fill_(7.0)
        lb.kv8_attention(q, cache, G.i32(table), G.i32(pos), out=out)
        assert not out[torch.from_numpy(at < 0).cuda()].any()
        G.check(out, ref, mag, size, dt, d, 300)
    assert K.device_status(reset=True) == 0
    far = np.where(pos < 0, 2000, pos)  # rows past the table, whose window is past it too
    ref, mag, size = R.attention(pool, q.double().cpu().numpy(), table, np.where(pos < 0, -1000, pos), window=40)
    for _ in range(20):
        out.fill_(7.0)
        lb.kv8_attention(q, cache, G.i32(table), G.i32(far), window=40, out=out)
        assert not out[torch.from_numpy(np.repeat(pos < 0, new)).cuda()].any()
        G.check(out, ref, mag, size, dt, d, 300)
    assert K.device_status(reset=True) == G.ERR_PAGE


def test_tiles_of_padding_take_the_prompt_kernel():
    cache = lb.KV8Cache.empty(60, 4, 64, page=64)
    q, table, pos = torch.ones((12 * 150, 8, 64), device="cuda"), G.i32(np.arange(60).reshape(12, 5)), G.i32([-150] * 12)
    lb.kv8_attention(q, cache, table, pos)
    assert "prompt_kernel" in G.kernels_of(lambda: lb.kv8_attention(q, cache, table, pos))
