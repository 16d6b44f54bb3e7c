"""The paged cache's places: pages that a sequence does not own are never written."""
import numpy as np
import pytest
import torch

import lowbit_b200 as lb
from lowbit_b200 import kernels as K
from lowbit_b200 import model as PM
from lowbit_b200.kvcache import PagedKVCache

pytestmark = pytest.mark.gpu
ERR_PAGE = -8


def bits(c):
    return [getattr(lay, n).clone() for lay in c.layers for n in ("k", "v", "k_exp", "v_exp")]


def step(c, cos, sin, gen, heads=4):
    """One token of every place through layer 0; the sequences' positions advance."""
    lay = c.layers[0]
    x = torch.randn((c.batch, (heads + 2 * lay.kv_heads) * lay.head_dim), generator=gen, device="cuda")
    q = lb.kv8_append(x, lay, c.table, c.pos, cos, sin)
    out = lb.kv8_attention(q, lay, c.table, c.pos)
    c.pos.add_(c.pos >= 0)
    return x, out


def test_a_released_place_writes_nowhere():
    cfg = PM.tiny_config()
    cos, sin = (torch.from_numpy(t).cuda() for t in PM.rope_tables(cfg.head_dim, 64, 1e4))
    c = PagedKVCache(cfg, 64, batch=3, page=16, pages=7)
    gen = torch.Generator(device="cuda").manual_seed(1)
    K.device_status(reset=True)
    c.reserve([20, 16, 1])
    c.set_lengths([19, 15, 0])
    step(c, cos, sin, gen)
    c.release(0)
    assert c.pos.tolist() == [-1, 16, 1] and c.table[0].tolist() == [-1] * 4 and c.lengths[0] == 0
    c.reserve([None, 48, 48])
    assert c.pos.tolist() == [-1, 16, 1] and c.table[0].tolist() == [-1] * 4
    assert not set(c._free) & set(c.table.flatten().tolist())
    alone = [t.clone() for t in (c.layers[0].k, c.layers[0].v, c.layers[0].k_exp, c.layers[0].v_exp)]
    x, out = step(c, cos, sin, gen)
    assert c.pos.tolist() == [-1, 17, 2] and K.device_status(reset=True) == 0 and not out[0].any()
    # the other two sequences without the free place: the same bits
    ref = lb.KV8Cache(*alone)
    q = lb.kv8_append(x[1:], ref, c.table[1:].contiguous(), torch.tensor([16, 1], dtype=torch.int32, device="cuda"), cos, sin)
    assert torch.equal(lb.kv8_attention(q, ref, c.table[1:].contiguous(), torch.tensor([16, 1], dtype=torch.int32, device="cuda")), out[1:])
    for n in ("k", "v", "k_exp", "v_exp"):
        assert torch.equal(getattr(c.layers[0], n), getattr(ref, n))
    c.set_lengths([0, 17, 2])
    assert c.pos.tolist() == [-1, 17, 2]
    c.reserve([5, 17, 2])
    assert c.pos.tolist() == [0, 17, 2] and c.table[0, 0] >= 0 and (c.table[0, 1:] == -1).all()


def test_tokens_without_a_page_are_recorded_and_not_stored():
    """A step past the reserved pages, and a place reserved for no tokens: skipped, no other page changes."""
    cfg = PM.tiny_config()
    cos, sin = (torch.from_numpy(t).cuda() for t in PM.rope_tables(cfg.head_dim, 64, 1e4))
    c = PagedKVCache(cfg, 64, batch=2, page=16, pages=4)
    gen = torch.Generator(device="cuda").manual_seed(2)
    K.device_status(reset=True)
    before = bits(c)
    step(c, cos, sin, gen)  # nothing is reserved
    assert K.device_status(reset=True) == ERR_PAGE and all(torch.equal(a, b) for a, b in zip(before, bits(c)))
    c.reserve([16, 0])
    c.set_lengths([16, 0])
    before = bits(c)
    step(c, cos, sin, gen)
    assert K.device_status(reset=True) == ERR_PAGE and all(torch.equal(a, b) for a, b in zip(before, bits(c)))


@pytest.mark.parametrize("graph", [True, False])
def test_a_place_is_used_again(graph):
    """Release one of three sequences and go on: the new one's tokens and the others' are those of fresh caches; a
    free place stays free over decode steps."""
    cfg = PM.tiny_config()
    m = PM.Model(cfg, PM.random_weights(cfg, seed=6), backend="w4a16")
    prompts = [[(i * k + 1) % 97 for i in range(n)] for k, n in ((3, 20), (5, 33), (7, 9))]
    c = m.new_cache(96, batch=3, kind="kv8", page=16)
    first = m.generate_ragged(prompts, 5, cache=c, graph=graph)
    c.release(1)
    tok = torch.tensor([first[0][-1], 0, first[2][-1]], device="cuda")
    c.reserve([25, None, 14])
    before = c.pos.tolist()
    m._step(tok, c)
    assert c.pos.tolist() == [before[0] + 1, -1, before[2] + 1]
    c.set_lengths([25, 0, 14])
    turn = [[1, 2], [9, 8, 7, 6], [5]]
    K.device_status(reset=True)
    got = m.generate_ragged(turn, 4, cache=c, graph=graph)
    assert K.device_status(reset=True) == 0 and c.lengths == [30, 7, 18] and c.pos.tolist() == c.lengths
    assert got[1] == m.generate(turn[1], 4, cache=m.new_cache(96, kind="kv8", page=16), graph=graph)
    for b in (0, 2):
        one = m.new_cache(96, kind="kv8", page=16)
        assert m.generate(prompts[b], 6, cache=one, graph=graph)[:5] == first[b]
        # the last token of the six was not appended, the sixth step's input was: the histories agree
        assert one.length == len(prompts[b]) + 5
        assert m.generate(turn[b], 4, cache=one, graph=graph) == got[b]


def test_lengths_stop_at_the_rotation_tables():
    """A cache may be longer than the model's positions, its sequences may not."""
    cfg = PM.tiny_config(max_position=40)
    m = PM.Model(cfg, PM.random_weights(cfg, seed=6), backend="fp32")
    K.device_status(reset=True)
    c = m.new_cache(100, batch=2, kind="kv8", page=16)
    got = m.generate_ragged([[1, 2, 3], [4] * 36], 5, cache=c)  # the fifth token is not appended
    assert c.lengths == [7, 40] and len(got[1]) == 5
    for call in (lambda: m.generate_ragged([[1], [2]], 1, cache=c), lambda: c.reserve([1, 41]),
                 lambda: m.generate_ragged([[1] * 38], 4), lambda: m.generate([1] * 38, 4, cache=m.new_cache(64, kind="kv8")),
                 lambda: m.forward([1] * 41, m.new_cache(64, kind="kv8"))):
        with pytest.raises(ValueError, match="max_position"):
            call()
    assert c.lengths == [7, 40] and K.device_status(reset=True) == 0
    m.forward([1] * 40, m.new_cache(64, kind="kv8"))
    assert K.device_status(reset=True) == 0


@pytest.mark.parametrize("n_new", [0, 1, 3])
def test_generate_batch_gives_whole_numbers(n_new):
    cfg = PM.tiny_config()
    m = PM.Model(cfg, PM.random_weights(cfg, seed=6), backend="fp32")
    prompts = np.arange(8).reshape(2, 4)
    a = m.generate_batch(prompts, n_new, cache=m.new_cache(16, batch=2))
    b = m.generate_batch(prompts, n_new, cache=m.new_cache(16, batch=2, kind="kv8"))
    assert a.dtype == b.dtype == np.int64 and a.shape == b.shape == (2, n_new)
