"""Edges of the paged 8-bit KV cache: tiles of padding, value scales far apart,
queries that are not finite, limits of the calls. Helpers, bounds and the
oracle are test_kv8_gpu.py's. With two KV heads and 100 rows a sequence, 12
sequences take the few-row kernel, 24 the prompt kernel."""
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
    zeros every time, and the other rows are right. (Twelve such sequences take the prompt kernel.)"""
    rng = np.random.default_rng(40)
    b, new, page = 12, 150, 64
    pool = G.host_pool(rng, 5 * b, 4, page, d)
    cache, table = G.device_pool(pool), rng.permutation(5 * b).reshape(b, 5)
    pos = np.array([0, -150, 70, -1000, 33, -130, 7, -149, 100, -150, 150, -64])
    q = torch.randn((b * new, 8, d), device="cuda").to(G.TYPES[dt])
    at = (pos[:, None] + np.arange(new)).reshape(-1)
    ref, mag, size, _ = attention(pool, q.double().cpu().numpy(), table, pos)
    out = torch.empty_like(q)
    for _ in range(20):
        out.fill_(7.0)
        lb.kv8_attention(q, cache, G.i32(table), G.i32(pos), out=out)
        assert not out[torch.from_numpy(at < 0).cuda()].any()
        G.check(out, ref, mag, size, dt, d, 300)
    assert K.device_status(reset=True) == 0
    far = np.where(pos < 0, 2000, pos)  # rows past the table, whose window is past it too
    ref, mag, size, _ = attention(pool, q.double().cpu().numpy(), table, np.where(pos < 0, -1000, pos), window=40)
    for _ in range(20):
        out.fill_(7.0)
        lb.kv8_attention(q, cache, G.i32(table), G.i32(far), window=40, out=out)
        assert not out[torch.from_numpy(np.repeat(pos < 0, new)).cuda()].any()
        G.check(out, ref, mag, size, dt, d, 300)
    assert K.device_status(reset=True) == G.ERR_PAGE


# ---------------------------------------------------------------- value scales far apart

def attention(pool, q, table, pos, window=0, scale=None):
    """R.attention in torch, 64 bits, for equal row counts (the same formulas, a sequence at a time), and
    max_i p_i 2^b_i times 127 times the number of visible tokens, b the value exponents [N, H, 1]."""
    kv, page, d = pool["k"].shape[1:]
    n, heads = q.shape[:2]
    new, g = n // len(pos), heads // kv
    scale = 1.0 / d ** 0.5 if scale is None else scale
    parts = []
    for i, p0 in enumerate(pos):
        at = p0 + torch.arange(new, device="cuda")
        length = max(1, int(p0) + new)
        ids = table[i, :-(-length // page)]
        x = torch.from_numpy(q[i * new:(i + 1) * new]).cuda().view(new, kv, g, d)
        k, v = (torch.from_numpy((pool[m][ids] * R.pow2(pool[m + "_exp"][ids])[..., None, None]).transpose(1, 0, 2, 3)
                                 .reshape(kv, -1, d)[:, :length]).cuda() for m in "kv")
        b = torch.from_numpy(R.pow2(pool["v_exp"][ids]).repeat(page, 0)[:length].T.copy()).cuda()
        j = torch.arange(length, device="cuda")
        seen = ((j <= at[:, None]) & ((j > at[:, None] - window) if window else True))[:, None, None]
        none = ~seen.any(-1)
        p = (scale * torch.einsum("tkgd,kld->tkgl", x, k)).masked_fill(~seen, -torch.inf).softmax(-1)
        p = p.masked_fill(none[..., None], 0.0)
        size = (scale * torch.einsum("tkgd,kld->tkgl", x.abs(), k.abs())).masked_fill(~seen, 0.0).amax(-1)
        floor = (p * b[None, :, None]).amax(-1, keepdim=True) * 127 * seen.sum(-1, keepdim=True)
        parts.append([y.reshape(new, heads, *y.shape[3:]).cpu().numpy() for y in (
            torch.einsum("tkgl,kld->tkgd", p, v), torch.einsum("tkgl,kld->tkgd", p, v.abs()), size, floor)])
    return [np.concatenate(y) for y in zip(*parts)]


def test_the_two_oracles_agree():
    rng = np.random.default_rng(39)
    pool = G.host_pool(rng, 12, 2, 16, 32)
    table, q = rng.permutation(12).reshape(3, 4), rng.standard_normal((15, 4, 32))
    for window in (0, 7):
        for a, b in zip(R.attention(pool, q, table, [-3, 0, 50], window=window), attention(pool, q, table, [-3, 0, 50], window)):
            np.testing.assert_allclose(a, b, rtol=1e-12, atol=1e-15)


def check(out, pool, q, table, pos, window, dt, d):
    """test_kv8_gpu.check with what weights held in fp16 lose at their lower end: half a subnormal step, 2^-25, where the
    row's largest p_i 2^b_i (b: the value exponent) stands for 2^13 or more: at most 2^-38 of it a code."""
    ref, mag, size, floor = attention(pool, q, table, pos, window)
    u, longest = 2.0 ** -22, max(pos) + len(q) // len(pos)
    tol = mag * ((2 * (d + 8) * size[..., None] + longest + 16) * u + G.R_P[dt]) + floor * 2.0 ** -38
    err = np.abs(out.double().cpu().numpy() - ref)
    assert np.isfinite(err).all()
    assert (err <= tol + np.maximum(G.R_OUT[dt] * np.abs(ref), G.TINY[dt])).all()


def far_case(dt, pos, new, low, gap, page, d, window=0, steer=False, b=1):
    """Value blocks of the pages `low` (a table slot, or a list of them) 2^gap below the others. `steer`: keys and
    queries that put the weight on those."""
    rng = np.random.default_rng(41)
    width = -(-(max(pos) + new) // page)
    pool = G.host_pool(rng, b * width, 2, page, d, 0.0)
    table = rng.permutation(b * width).reshape(b, width)
    pool["v_exp"] = (pool["v_exp"].astype(int) + 60 * (gap > 110)).astype(np.uint8)
    ids = table[:, np.atleast_1d(low)]
    pool["v_exp"][ids] -= gap
    q = rng.standard_normal((b * new, 4, d))
    if steer:
        pool["k"] = -np.abs(pool["k"])
        pool["k"][ids] = np.abs(pool["k"][ids])
        q = np.abs(q) * 4
    q = torch.from_numpy(q.astype(np.float32)).to(G.TYPES[dt])
    out = lb.kv8_attention(q.cuda(), G.device_pool(pool), G.i32(table), G.i32(pos), window=window)
    check(out, pool, q.double().numpy(), table, pos, window, dt, d)
    assert K.device_status(reset=True) == 0


GAPS = [40, 59, 62, 75, 110, 170]


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("page,d", [(16, 32), (32, 64), (64, 128)])
def test_rows_that_see_small_values_only(dt, gap, page, d):
    """Later, larger tokens do not change a row that does not see them: few rows, prompts, windows."""
    far_case(dt, [page - 2], 5, 0, gap, page, d)                # the first rows end inside the small block
    far_case(dt, [2 * page - 3], 6, 1, gap, page, d, window=2)  # some rows' windows hold small tokens only
    for b in (12, 24):  # the few-row kernel, the prompt kernel
        far_case(dt, [0] * b, 100, 0, gap, page, d, b=b)
        far_case(dt, [3] * b, 140, [1, 2], gap, page, d, window=9, b=b)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("new,b", [(1, 1), (5, 3), (100, 12), (100, 24)])
def test_weight_on_small_values(dt, gap, new, b):
    """Large values are seen, but the weight lies on small ones."""
    far_case(dt, [150] * b, new, [1, 3], gap, 32, 64, steer=True, b=b)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("new", [1, 2, 3])
@pytest.mark.parametrize("page,step", [(16, 10), (16, 4), (64, 1)])
def test_scales_that_rise_along_a_long_context(dt, new, page, step):
    """Each `step` pages twice the last ones' values, over enough sequences that a block of the grid looks pages up
    several times; windows that end anywhere. Within the bound of test_kv8_gpu.check, which is relative to the row."""
    rng = np.random.default_rng(42)
    kv, d, b, length, window = 8, 32, 64, 8192, 700
    n = length // page
    pool = G.host_pool(rng, n, kv, page, d, 0.0)
    pool["v_exp"] = (20 + np.arange(n)[:, None] // step + 0 * pool["v_exp"]).astype(np.uint8)
    table = np.broadcast_to(np.arange(n), (b, n))
    pos = np.linspace(window, length - new, b).astype(int)
    q = torch.randn((b * new, kv, d), device="cuda").to(G.TYPES[dt])
    k, v = (torch.from_numpy((pool[m] * R.pow2(pool[m + "_exp"])[..., None, None]).transpose(1, 0, 2, 3).reshape(kv, length, d)).cuda()
            for m in "kv")
    at = (torch.from_numpy(pos).cuda()[:, None] + torch.arange(new, device="cuda")).view(-1, 1)
    j = torch.arange(length, device="cuda")
    s = torch.einsum("rhd,hld->rhl", q.double(), k) / d ** 0.5
    size = torch.einsum("rhd,hld->rhl", q.double().abs(), k.abs()).amax(-1) / d ** 0.5
    for win in (0, window):
        seen = (j <= at) & ((j > at - win) if win else True)
        p = s.masked_fill(~seen[:, None], -torch.inf).softmax(-1)
        ref, mag = torch.einsum("rhl,hld->rhd", p, v), torch.einsum("rhl,hld->rhd", p, v.abs())
        out = lb.kv8_attention(q, G.device_pool(pool), G.i32(table), G.i32(pos), window=win)
        G.check(out, ref.cpu().numpy(), mag.cpu().numpy(), size.cpu().numpy(), dt, d, length)


@pytest.mark.parametrize("new,b", [(1, 1), (100, 12), (100, 24)])
def test_largest_and_smallest_values_together(new, b):
    """Values near the type's end beside ones 2^200 below: sums stay finite."""
    rng = np.random.default_rng(43)
    pool = G.host_pool(rng, 8 * b, 2, 32, 64, 0.0)
    pool["v"] = np.clip(pool["v"], -63, 63)
    table = rng.permutation(8 * b).reshape(b, 8)
    pool["v_exp"][:] = 249
    pool["v_exp"][table[:, ::2]] = 49
    q = rng.standard_normal((b * new, 4, 64)).astype(np.float32)
    pos = [256 - new] * b
    out = lb.kv8_attention(torch.from_numpy(q).cuda(), G.device_pool(pool), G.i32(table), G.i32(pos))
    G.check(out, *attention(pool, q.astype(np.float64), table, pos)[:3], "fp32", 64, 256)


@pytest.mark.parametrize("dt", G.TYPES)
@pytest.mark.parametrize("new,b", [(3, 2), (100, 12), (100, 24)])
def test_far_scales_with_bad_places(dt, new, b):
    """Where the scales are far apart too: a NaN block spoils the rows that see it, a missing page is left out."""
    rng = np.random.default_rng(44)
    page, d, w = 16, 64, 10
    pool = G.host_pool(rng, b * w, 2, page, d, 0.0)
    table = rng.permutation(b * w).reshape(b, w)
    pool["v_exp"][table[:, 1]] -= 80
    pool["v_exp"][table[0, 4], 1] = 255
    p0 = 5 * page - new // 2
    pos = [p0] * b
    q = torch.randn((b * new, 4, d), device="cuda").to(G.TYPES[dt])
    cache = G.device_pool(pool)
    out = lb.kv8_attention(q, cache, G.i32(table), G.i32(pos), window=200).float().cpu().numpy().reshape(b, new, 4, d)
    sees = p0 + np.arange(new) >= 4 * page
    assert np.isnan(out[0, sees, 2:]).all() and np.isfinite(out[0, ~sees]).all()
    assert np.isfinite(out[0, :, :2]).all() and np.isfinite(out[1:]).all()
    clean = {n: a.copy() for n, a in pool.items()}
    clean["v_exp"][table[0, 4], 1] = 121
    K.device_status(reset=True)
    bad = table.copy()
    bad[1, 3] = -1
    out = lb.kv8_attention(q, G.device_pool(clean), G.i32(bad), G.i32(pos))
    assert K.device_status(reset=True) == G.ERR_PAGE
    # leaving page 3 out is a row over the remaining tokens
    keep = np.r_[0:3 * page, 4 * page:w * page]
    k, v = (torch.from_numpy((clean[n][table[1]] * R.pow2(clean[n + "_exp"][table[1]])[..., None, None])
                             .transpose(1, 0, 2, 3).reshape(2, w * page, d)).cuda() for n in "kv")
    x = q.double().view(b, new, 2, 2, d)[1]
    s = torch.einsum("tkgd,kld->tkgl", x, k) / d ** 0.5
    size = torch.einsum("tkgd,kld->tkgl", x.abs(), k.abs()).amax(-1) / d ** 0.5
    at = p0 + torch.arange(new, device="cuda")[:, None]
    j = torch.arange(w * page, device="cuda")
    seen = (j <= at) & torch.isin(j, torch.from_numpy(keep).cuda())
    p = s.masked_fill(~seen[:, None, None], -torch.inf).softmax(-1)
    ref, mag = torch.einsum("tkgl,kld->tkgd", p, v), torch.einsum("tkgl,kld->tkgd", p, v.abs())
    G.check(out.view(b, new, 4, d)[1], *(t.reshape(new, 4, -1).squeeze(-1).cpu().numpy() for t in (ref, mag, size)), dt, d, w * page)


@pytest.mark.parametrize("dt", G.TYPES)
@pytest.mark.parametrize("new,b,length", [(1, 1, 500), (1, 1, 60000), (3, 40, 900), (100, 12, 300), (100, 24, 300)])
def test_scores_past_2_to_24(dt, new, b, length):
    """Scores so large that whole numbers are no longer exact in fp32: a row stays between its smallest and largest
    visible value (a factor 2 of the softmax's references would leave that range)."""
    rng = np.random.default_rng(45)
    page = 64
    width = -(-length // page)
    pool = G.host_pool(rng, width, 2, page, 64)
    pool["v"] = np.maximum(np.abs(pool["v"]), 32).astype(np.int8)  # a block's values lie within a factor 4
    table = np.broadcast_to(np.arange(width), (b, width))
    q = torch.randn((b * new, 4, 64), device="cuda").to(G.TYPES[dt])
    cache, v = G.device_pool(pool), pool["v"] * R.pow2(pool["v_exp"])[..., None, None]
    lo, hi = v.min((0, 2)).repeat(2, 0), v.max((0, 2)).repeat(2, 0)  # by query head
    for scale in 2.0 ** np.arange(16, 64, 1.5):
        out = lb.kv8_attention(q, cache, G.i32(table), G.i32([length - new] * b), scale=scale).double().cpu().numpy()
        assert (out >= lo * (1 - 2.0 ** -8)).all() and (out <= hi * (1 + 2.0 ** -8)).all(), scale


@pytest.mark.parametrize("dt", G.TYPES)
@pytest.mark.parametrize("new,b", [(1, 1), (1, 40), (3, 2), (100, 12), (100, 24)])
def test_infinite_queries(dt, new, b):
    """softmax of infinite scores is NaN, whatever their signs; a row that sees nothing is 0 whatever its query;
    other rows are as without them."""
    rng = np.random.default_rng(46)
    pool = G.host_pool(rng, 8, 2, 64, 64)
    table = np.broadcast_to(np.arange(8), (b, 8))
    q = torch.randn((b * new, 4, 64), device="cuda").to(G.TYPES[dt])
    for sign in (1, -1):  # keys that are all positive make scores of one sign
        pool["k"] = (sign * np.maximum(np.abs(pool["k"]), 1)).astype(np.int8)
        cache = G.device_pool(pool)
        for p0 in (0, 300, -1, -new):
            pos = G.i32([p0] * b)
            ref = lb.kv8_attention(q, cache, G.i32(table), pos)
            for bad in (float("inf"), float("-inf"), float("nan")):
                x = q.clone()
                x[0, 1, 5] = x[-1, 3, 63] = bad
                for scale in (None, 0.0):
                    out = lb.kv8_attention(x, cache, G.i32(table), pos, scale=scale)
                    base = ref if scale is None else lb.kv8_attention(q, cache, G.i32(table), pos, scale=scale)
                    hit = torch.zeros((b * new, 4), dtype=torch.bool, device="cuda")
                    hit[0, 1] = hit[-1, 3] = True
                    sees = torch.from_numpy((p0 + np.arange(new) >= 0)[None].repeat(b, 0).reshape(-1)).cuda()
                    nan = hit & sees[:, None]
                    assert torch.isnan(out[nan]).all() and not out[~sees].any()
                    # (a row's references follow votes of rows beside it: other roundings, the same value)
                    torch.testing.assert_close(out[~nan].float(), base[~nan].float(), rtol=2 * G.R_OUT[dt] + 2.0 ** -10, atol=2.0 ** -10)


@pytest.mark.parametrize("heads", [4, 128])
@pytest.mark.parametrize("b", [2, 40])
def test_rows_left_out_by_max_tokens_are_recorded(heads, b):
    """max_tokens below the rows of a sequence, 0 included: the rows left out are not written, and recorded."""
    rng = np.random.default_rng(47)
    pool = G.host_pool(rng, 8, 2, 64, 64)
    table, pos = G.i32(np.broadcast_to(np.arange(8), (b, 8))), G.i32([100] * b)
    q = torch.randn((2 * b, heads, 64), device="cuda")
    cos, sin = (torch.from_numpy(t).cuda() for t in G.rope_tables(64, 512, 1e4))
    qkv = torch.randn((2 * b, (heads + 4) * 64), device="cuda")
    starts, none = G.i32(np.arange(b + 1) * 2), G.i32([0] * (b + 1))
    for most in (0, 1):
        cache = G.device_pool(pool)
        out = lb.kv8_attention(q, cache, table, pos, starts=starts, max_tokens=most, out=torch.full_like(q, 7.0))
        assert K.device_status(reset=True) == G.ERR_PAGE
        left = out.view(b, 2, heads, 64)[:, most:]
        assert (left == 7).all() and torch.isfinite(out).all()
        lb.kv8_append(qkv, cache, table, pos, cos, sin, starts=starts, max_tokens=most)
        assert K.device_status(reset=True) == G.ERR_PAGE
        if most == 0:
            G.same_pool(cache, pool)
        # no sequence has rows: nothing to leave out
        lb.kv8_attention(q, cache, table, pos, starts=none, max_tokens=most)
        lb.kv8_append(qkv, cache, table, pos, cos, sin, starts=none, max_tokens=most)
        assert K.device_status(reset=True) == 0


# A quarter of half an ulp: what the sums may drift by before a total is kept, and with one
DRIFT = {"fp16": 2.0 ** -13, "bf16": 2.0 ** -10}


@pytest.mark.parametrize("dt,new,b,kv,g,d,page,length", [
    ("fp16", 100, 12, 2, 4, 128, 64, 8192), ("fp16", 100, 12, 2, 4, 128, 64, 131072), ("fp16", 90, 12, 4, 2, 64, 32, 70001),
    ("fp16", 100, 12, 4, 2, 32, 128, 131072), ("bf16", 100, 12, 2, 4, 128, 64, 131072), ("bf16", 100, 12, 2, 4, 128, 64, 1 << 20),
    ("fp16", 1, 148, 4, 2, 64, 64, 16384), ("fp16", 1, 64, 4, 2, 64, 64, 131072), ("fp16", 3, 64, 4, 4, 128, 16, 131071),
    ("fp16", 5, 64, 4, 4, 32, 128, 131072), ("bf16", 1, 32, 2, 8, 128, 64, 1 << 20), ("bf16", 2, 40, 2, 8, 64, 32, 300001)])
def test_long_sums_of_16_bit_types_do_not_drift(dt, new, b, kv, g, d, page, length):
    """Positive values, so that truncated sums would come out small: the mean error beyond that of the correctly
    rounded rows stays within DRIFT, at any length."""
    pages = -(-length // page)
    cache = lb.KV8Cache.empty(pages, kv, d, page=page)
    cache.k.copy_(torch.randint(-60, 61, cache.k.shape, device="cuda"))
    cache.v.copy_(torch.randint(32, 97, cache.v.shape, device="cuda"))
    cache.k_exp.fill_(122)
    cache.v_exp.fill_(121)
    table = torch.randperm(pages, device="cuda").to(torch.int32)
    tables = table[None].repeat(b, 1)  # one prefix for all
    q = torch.randn((b * new, kv * g, d), device="cuda").to(G.TYPES[dt])
    out = lb.kv8_attention(q, cache, tables, G.i32([length - new] * b))
    again = lb.kv8_attention(q, cache, tables, G.i32([length - new] * b))
    assert torch.equal(out, again)
    rows = torch.arange(0, b * new, max(1, b * new // 24), device="cuda")
    at = length - new + rows % new
    e = []
    for h in range(kv):
        k, v = (t[table.long(), h].reshape(-1, d)[:length].double() for t in (cache.k, cache.v))
        x = q[rows, h * g:(h + 1) * g].double()
        s = (x @ (k.T * 2.0 ** -5) / d ** 0.5).masked_fill((torch.arange(length, device="cuda") > at[:, None])[:, None], -torch.inf)
        ref = s.softmax(-1) @ v * 2.0 ** -6
        e.append(((out[rows, h * g:(h + 1) * g].double() - ref.to(G.TYPES[dt]).double()) / ref).mean().item())
    assert abs(np.mean(e)) <= DRIFT[dt], np.mean(e)


@pytest.mark.parametrize("new,b", [(1, 40), (3, 20), (100, 24)])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_fp16_weights_keep_22_bits(new, b, d):
    """fp16 calls hold weights in two fp16 pieces. Few tokens and small scores, so that the bound of test_kv8_gpu.check
    is narrow enough with r_p = 2^-21 (two pieces, as its fp32) to exclude weights of one piece (11 bits), which the
    oracle shows with such weights planted in it."""
    rng = np.random.default_rng(48)
    pool = G.host_pool(rng, 2 * b + 8, 2, 64, d, 0.2)
    table = np.stack([rng.permutation(2 * b + 8)[:4] for _ in range(b)])
    q = torch.from_numpy(rng.standard_normal((b * new, 4, d)).astype(np.float32)).to(torch.float16)
    pos, window, scale = [70] * b, 12, 0.08 / d
    out = lb.kv8_attention(q.cuda(), G.device_pool(pool), G.i32(table), G.i32(pos), window=window, scale=scale)
    x = q.double().numpy()
    ref, mag, size, _ = attention(pool, x, table, pos, window, scale)
    tol = mag * ((2 * (d + 8) * size[..., None] + window + 16) * 2.0 ** -22 + 2.0 ** -21)
    tol += np.maximum(G.R_OUT["fp16"] * np.abs(ref), G.TINY["fp16"])
    assert (np.abs(out.double().cpu().numpy() - ref) <= tol).all()
    one = np.zeros_like(ref)  # the same with weights rounded to 11 bits
    for i in range(b * new):
        p = 70 + i % new
        at = np.arange(p - window + 1, p + 1)
        ids = table[i // new, at // 64]
        for h in range(4):
            g = h // 2
            k = pool["k"][ids, g, at % 64] * R.pow2(pool["k_exp"][ids, g])[:, None]
            t = scale * (k @ x[i, h]) / np.log(2) + pool["v_exp"][ids, g] - 127.0
            w = np.exp2(t - np.ceil(t.max()) + 14)
            w16 = w.astype(np.float16).astype(np.float64)
            l = (w / R.pow2(pool["v_exp"][ids, g])).sum()
            one[i, h] = w16 @ pool["v"][ids, g, at % 64] / l
            assert np.allclose(w @ pool["v"][ids, g, at % 64] / l, ref[i, h], rtol=1e-9, atol=1e-9)
    assert (np.abs(one - ref) > tol).mean() > 0.01


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_totals_of_ragged_prompts(dt):
    """Contexts long enough for totals in the workspace, sequences of very different numbers of rows, tiles that end
    inside: the rows of equal prompts one by one, and a workspace that goes by the rows, not by sequences times rows."""
    kv, g, d, page, length = 2, 4, 64, 64, 10000 if dt == "fp16" else 140000
    pages = -(-length // page)
    cache = lb.KV8Cache.empty(pages, kv, d, page=page)
    cache.k.copy_(torch.randint(-60, 61, cache.k.shape, device="cuda"))
    cache.v.copy_(torch.randint(-96, 97, cache.v.shape, device="cuda"))
    cache.k_exp.fill_(122)
    cache.v_exp.fill_(121)
    table = torch.randperm(pages, device="cuda").to(torch.int32)
    new = [1, 70, 0, 200, 33, 129, 64, 300, 5, 90, 128, 150]
    b, n = len(new), sum(new)
    starts = np.concatenate([[0], np.cumsum(new)])
    pos = [length - t for t in new]
    q = torch.randn((n, kv * g, d), device="cuda").to(G.TYPES[dt])
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.max_memory_allocated()
    out = lb.kv8_attention(q, cache, table[None].repeat(b, 1), G.i32(pos), starts=G.i32(starts))  # max_tokens left to N
    assert torch.cuda.max_memory_allocated() - before < 8 * n * kv * g * d * 4 + (1 << 20)
    same = lb.kv8_attention(q, cache, table[None].repeat(b, 1), G.i32(pos), starts=G.i32(starts), max_tokens=300)
    assert torch.equal(out, same)
    k, v = (t[table.long()].transpose(0, 1).reshape(kv, -1, d)[:, :length].double() * 2.0 ** e
            for t, e in ((cache.k, -5), (cache.v, -6)))
    at = torch.from_numpy(np.concatenate([np.arange(p, p + t) for p, t in zip(pos, new)])).cuda()
    for i in list(range(0, n, 37)) + [n - 1]:
        x = q[i].double().view(kv, g, d)
        s = (torch.einsum("kgd,kld->kgl", x, k) / d ** 0.5)[..., :at[i] + 1]
        ref = torch.einsum("kgl,kld->kgd", s.softmax(-1), v[:, :at[i] + 1]).view(kv * g, d)
        mag = torch.einsum("kgl,kld->kgd", s.softmax(-1), v[:, :at[i] + 1].abs()).view(kv * g, d)
        size = (torch.einsum("kgd,kld->kgl", x.abs(), k.abs()).amax(-1) / d ** 0.5).view(kv * g)
        G.check(out[i], ref.cpu().numpy(), mag.cpu().numpy(), size.cpu().numpy(), dt, d, length)


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("new,b,page,length", [(1, 1, 16, 700), (1, 2, 64, 300), (5, 3, 32, 500), (100, 12, 64, 1500), (130, 12, 16, 1100), (100, 24, 64, 1300)])
@pytest.mark.parametrize("where", ["first", "last", "mixed"])
@pytest.mark.parametrize("tiny", [False, True])
def test_blocks_of_exponent_0(dt, new, b, page, length, where, tiny):
    """All-zero value blocks before, behind and among ordinary ones (a cache that was not filled) count in the softmax;
    blocks of exponent 0 with codes are values of 2^-127 a code, and rows that see only those get them."""
    rng = np.random.default_rng(49)
    width = -(-length // page)
    pool = G.host_pool(rng, b * width, 2, page, 64, 0.3)
    table = rng.permutation(b * width).reshape(b, width)
    o = {"first": range(width - 1), "last": range(1, width), "mixed": range(0, width, 3)}[where]
    ids = table[:, list(o)].ravel()
    pool["v_exp"][ids] = 0
    if not tiny:
        pool["v"][ids] = 0
    q = torch.from_numpy(rng.standard_normal((b * new, 4, 64)).astype(np.float32)).to(G.TYPES[dt])
    for pos, window in ((length - new, 0), (length - new, 40), (0, 0)):
        out = lb.kv8_attention(q.cuda(), G.device_pool(pool), G.i32(table), G.i32([pos] * b), window=window)
        check(out, pool, q.double().numpy(), table, [pos] * b, window, dt, 64)


@pytest.mark.parametrize("new,b", [(1, 200), (3, 150)])
def test_zeros_before_values_in_a_long_segment(new, b):
    """The zeros end after several lookups of a block of the grid; the tokens behind them are the only values."""
    kv, d, length, page = 8, 32, 8192, 16
    rng = np.random.default_rng(50)
    n = length // page
    pool = G.host_pool(rng, n, kv, page, d)
    for first in (100, 300, 500):
        part = {m: a.copy() for m, a in pool.items()}
        part["v"][:first], part["v_exp"][:first] = 0, 0
        q = torch.randn((b * new, kv, d), device="cuda")
        out = lb.kv8_attention(q, G.device_pool(part), G.i32(np.broadcast_to(np.arange(n), (b, n))), G.i32([length - new] * b))
        k, v = (torch.from_numpy((part[m] * R.pow2(part[m + "_exp"])[..., None, None]).transpose(1, 0, 2, 3).reshape(kv, length, d)).cuda()
                for m in "kv")
        at = (length - new + torch.arange(new, device="cuda")).repeat(b)
        s = torch.einsum("rhd,hld->rhl", q.double(), k) / d ** 0.5
        size = torch.einsum("rhd,hld->rhl", q.double().abs(), k.abs()).amax(-1) / d ** 0.5
        p = s.masked_fill((torch.arange(length, device="cuda") > at[:, None])[:, None], -torch.inf).softmax(-1)
        G.check(out, *(t.cpu().numpy() for t in (torch.einsum("rhl,hld->rhd", p, v), torch.einsum("rhl,hld->rhd", p, v.abs()), size)),
                "fp32", d, length)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("new,b,length", [(1, 1, 20000), (1, 9, 3000), (4, 12, 1500), (100, 12, 1500)])
@pytest.mark.parametrize("gap", [45, 80, 120])
def test_far_scales_in_one_part_of_a_long_row(dt, new, b, length, gap):
    """The row is cut over the grid: parts with scales far apart, computed otherwise, join parts of large or of small
    values only; the weight lies where the values are small, or large, or anywhere."""
    rng = np.random.default_rng(51)
    page, d = 64, 64
    width = -(-length // page)
    pool = G.host_pool(rng, b * width, 2, page, d, 0.0)
    table = rng.permutation(b * width).reshape(b, width)
    small = table[:, :width * 3 // 4]
    pool["v_exp"][small] -= gap
    for weight in (0, 1, -1):
        part = {n: a.copy() for n, a in pool.items()}
        q = rng.standard_normal((b * new, 4, d))
        if weight:  # on the small values, or on the large ones
            part["k"] = -weight * np.abs(part["k"])
            part["k"][small] = weight * np.abs(part["k"][small])
            q = np.abs(q)
        q = torch.from_numpy(q.astype(np.float32)).to(G.TYPES[dt])
        for pos in ([length - new] * b, [width * 3 // 4 * page - 2] * b):
            out = lb.kv8_attention(q.cuda(), G.device_pool(part), G.i32(table), G.i32(pos))
            check(out, part, q.double().numpy(), table, pos, 0, dt, d)


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("new,b,page,length", [(1, 1, 64, 500), (1, 200, 16, 4100), (5, 3, 16, 1100), (100, 24, 64, 1300)])
@pytest.mark.parametrize("zeros", ["first", "last"])
def test_weight_on_blocks_of_zeros(dt, new, b, page, length, zeros):
    """The softmax lies on blocks of zeros, by 2^64: what is left of the values keeps its digits."""
    rng = np.random.default_rng(52)
    width, kv, d = -(-length // page), 2 if b < 200 else 8, 64
    pool = G.host_pool(rng, width, kv, page, d, 0.0)
    table = np.broadcast_to(rng.permutation(width), (b, width))
    ids = table[0, :width // 2] if zeros == "first" else table[0, width // 2:]
    pool["v"][ids], pool["v_exp"][ids] = 0, 0
    pool["k_exp"][:] -= 4
    pool["k"][ids], pool["k_exp"][ids] = 64, 122
    q = torch.from_numpy((2.775 + 0.01 * rng.standard_normal((b * new, 2 * kv, d))).astype(np.float32)).to(G.TYPES[dt])
    pos = [length - new] * b
    out = lb.kv8_attention(q.cuda(), G.device_pool(pool), G.i32(table), G.i32(pos))
    ref, mag, size, _ = attention(pool, q.double().numpy(), table, pos)
    assert 2.0 ** -70 < mag.max() < 2.0 ** -50
    if dt == "fp16":
        assert not out.any()
    else:
        G.check(out, ref, mag, size, dt, d, length)
