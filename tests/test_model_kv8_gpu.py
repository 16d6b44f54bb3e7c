"""The decoder over the paged 8-bit KV cache: against the numpy model whose
attention runs on the oracle's quantised cache, against itself in pieces, and
prompts of different lengths together.

Tolerance 1e-2 (as the W4A8 model's): linears that differ in their last bits
move single codes across a rounding boundary, one step (1/127 of a block's
largest value at most 2/127) of one key or value among many."""
import numpy as np
import pytest
import torch

from lowbit_b200 import kernels as K
from lowbit_b200 import model as PM
from lowbit_b200.kvcache import PagedKVCache
from oracle import kv8_ref as KR
from oracle import model_ref as O

pytestmark = pytest.mark.gpu


def rel(a, b):
    return float(np.abs(np.asarray(a, np.float64) - b).max() / np.abs(b).max())


class QuantisedCache:
    def __init__(self, cfg, max_len, page):
        n, kv, d = -(-max_len // page), cfg.num_kv_heads, cfg.head_dim
        self.pools = [{"k": np.zeros((n, kv, page, d), np.int8), "v": np.zeros((n, kv, page, d), np.int8),
                       "k_exp": np.zeros((n, kv), np.uint8), "v_exp": np.zeros((n, kv), np.uint8)}
                      for _ in range(cfg.num_layers)]
        self.table, self.length = np.arange(n)[None], 0


class QuantisedModel(O.Model):
    def _attention(self, q, k, v, cache, li, pos):
        t, h, d = q.shape
        rows = np.concatenate([a.reshape(t, -1) for a in (q, k, v)], 1)  # already rotated: angle 0
        one = np.ones((pos + t, d // 2), np.float32)
        KR.append(cache.pools[li], rows, cache.table, [pos], one, 0 * one, h)
        return KR.attention(cache.pools[li], q, cache.table, [pos])[0].reshape(t, h * d).astype(np.float32)


def pair(seed, **over):
    cfg = PM.tiny_config(**over)
    W = PM.random_weights(cfg, seed=seed)
    lin = {key: O.lin_fp32(w, b) for key, (w, b) in O.concat_weights(O.tiny_cfg(**over), W).items()}
    return PM.Model(cfg, W, backend="fp32"), QuantisedModel(O.tiny_cfg(**over), W, lin)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("over", [{}, dict(num_heads=8, num_kv_heads=1, head_dim=32), dict(head_dim=128, qkv_bias=False)])
def test_forward_matches_the_quantised_oracle(page, over):
    m, ref = pair(3, **over)
    toks = [(i * 13 + 5) % 97 for i in range(90)]
    cache, rc = m.new_cache(96, kind="kv8", page=page), QuantisedCache(m.cfg, 96, page)
    got = [m.forward(toks[:40], cache, logits="all"), m.forward(toks[40:75], cache, logits="all")]
    want = [ref.forward(toks[:40], rc, logits="all"), ref.forward(toks[40:75], rc, logits="all")]
    for t in toks[75:]:
        got.append(m.forward([t], cache)[None])
        want.append(ref.forward([t], rc)[None])
    assert cache.length == 90 and K.device_status(reset=True) == 0
    assert rel(np.concatenate(got), np.concatenate(want)) < 1e-2
    with pytest.raises(ValueError):
        m.forward([1] * 7, cache)


@pytest.mark.parametrize("backend", ["w4a16", "w4a8", "mxfp4", "fp32"])
def test_close_to_the_fp32_cache(backend):
    """Keys and values to 1/254 of a block's largest value at worst: logits within a few per cent."""
    cfg = PM.tiny_config()
    m = PM.Model(cfg, PM.random_weights(cfg, seed=4), backend=backend)
    toks = [(i * 7 + 3) % 97 for i in range(100)]
    a = m.forward(toks, m.new_cache(100), logits="all")
    b = m.forward(toks, m.new_cache(100, kind="kv8"), logits="all")
    assert rel(b, a) < 5e-2


@pytest.mark.parametrize("graph", [True, False])
def test_ragged_prompts_decode_as_alone(graph):
    cfg = PM.tiny_config()
    m = PM.Model(cfg, PM.random_weights(cfg, seed=6), backend="w4a16", asym=True)
    prompts = [[(i * k + 1) % 97 for i in range(n)] for k, n in ((3, 5), (5, 33), (7, 1), (11, 70))]
    got = m.generate_ragged(prompts, 9, graph=graph)
    for p, g in zip(prompts, got):
        assert g == m.generate(p, 9, cache=m.new_cache(len(p) + 9, kind="kv8"), graph=graph)
    assert K.device_status(reset=True) == 0


def test_equal_prompts_and_a_second_turn():
    cfg = PM.tiny_config()
    m = PM.Model(cfg, PM.random_weights(cfg, seed=8), backend="w4a16")
    prompts = (np.arange(3 * 9).reshape(3, 9) * 11) % cfg.vocab_size
    cache = m.new_cache(64, batch=3, kind="kv8", page=16)
    first = m.generate_batch(prompts, 6, cache=cache)
    assert first.shape == (3, 6) and cache.lengths == [14] * 3
    turn = [[1, 2, 3], [4], [5, 6]]
    more = m.generate_ragged(turn, 4, cache=cache)
    assert cache.lengths == [20, 18, 19] and cache.pos.tolist() == cache.lengths
    for b in range(3):  # the same conversation alone
        c = m.new_cache(64, kind="kv8", page=16)
        assert m.generate(prompts[b], 6, cache=c) == list(first[b])
        assert m.generate(turn[b], 4, cache=c) == more[b]


def test_pages_come_and_go():
    cfg = PM.tiny_config()
    c = PagedKVCache(cfg, 64, batch=3, page=16, pages=7)
    c.reserve([20, 16, 1])
    assert len(c._free) == 3 and c.capacity == 64 and c.nbytes == cfg.num_layers * c.layers[0].nbytes
    t = c.table.cpu()
    assert len({int(t[0, 0]), int(t[0, 1]), int(t[1, 0]), int(t[2, 0])}) == 4
    with pytest.raises(ValueError, match="out of pages"):
        c.reserve([64, 48, 16])
    with pytest.raises(ValueError, match="full"):
        c.reserve([65, 0, 0])
    with pytest.raises(ValueError):
        c.reserve([1, 2])
    assert torch.equal(c.table.cpu(), t)
    c.set_lengths([20, 16, 1])
    with pytest.raises(ValueError, match="different lengths"):
        c.length
    c.release(0)
    c.reserve([0, 48, 48])
    assert len(c._free) == 7 - 3 - 3 and c.lengths == [0, 16, 1] and c.pos.tolist() == [0, 16, 1]
    m = PM.Model(cfg, PM.random_weights(cfg, seed=1), backend="fp32")
    with pytest.raises(ValueError):
        m.new_cache(8, kind="fp8")
    with pytest.raises(ValueError):
        m.generate_ragged([[1], []], 2)
    with pytest.raises(ValueError):
        m.generate_ragged([[1], [2, 3]], 2, cache=m.new_cache(8, batch=2))
    with pytest.raises(ValueError):
        m.generate_ragged([[1]], 2, cache=m.new_cache(8, batch=2, kind="kv8"))
