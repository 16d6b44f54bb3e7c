"""Paged 8-bit KV cache on the GPU against the oracle (oracle/kv8_ref.py).

append and read are compared bit for bit. attention is compared within bounds
derived from its arithmetic, with u = 2^-22 (tensor cores align the products
of a step to its largest and truncate):
  a score sums D products:          |ds| <= (D + 8) u S, S = max_j scale sum_d |q_d k_jd|
  a weight p is off by 2 |ds| (its own score and the maximum's) plus a few ulps of exp2;
  sums over L keys add at most L u; 16-bit types round p once to 11 bits (2^-11);
so |d out| <= sum_j p_j |v_j| (2 (D + 8) u S + (L + 16) u + r_p) + r_out |out|, r_out the
output type's half ulp."""
import numpy as np
import pytest
import torch

import lowbit_b200 as lb
from lowbit_b200 import kernels as K
from lowbit_b200.model import rope_tables
from oracle import kv8_ref as R

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
R_P = {"fp32": 2.0 ** -21, "bf16": 2.0 ** -11, "fp16": 2.0 ** -11}
R_OUT = {"fp32": 2.0 ** -24, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
TINY = {"fp32": 2.0 ** -150, "bf16": 2.0 ** -134, "fp16": 2.0 ** -25}  # half ulp of subnormal outputs
ERR_PAGE = -8


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


def host_pool(rng, pages, kv, page, d, spread=0.5):
    p = {}
    for n in "kv":
        x = rng.standard_normal((pages, kv, page, d)) * np.exp(spread * rng.standard_normal((pages, kv, 1, 1)))
        e = np.vectorize(R.scale_byte)(np.abs(x).max((2, 3)))
        p[n] = np.rint(x / R.pow2(e)[..., None, None]).astype(np.int8)
        p[n + "_exp"] = e.astype(np.uint8)
    return p


def device_pool(p):
    return lb.KV8Cache(*(torch.from_numpy(p[n].copy()).cuda() for n in ("k", "v", "k_exp", "v_exp")))


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def tables(rng, counts, pages, junk=0):
    """A page table [B, width]: distinct pages in random order, `junk` ids past each sequence's own."""
    ids = rng.permutation(pages)
    t = np.full((len(counts), max(1, max(counts))), junk, np.int64)
    at = 0
    for b, c in enumerate(counts):
        t[b, :c] = ids[at:at + c]
        at += c
    return t


def check(out, ref, mag, size, dt, d, longest):
    u = 2.0 ** -22
    tol = mag * ((2 * (d + 8) * size[..., None] + longest + 16) * u + R_P[dt]) + np.maximum(R_OUT[dt] * np.abs(ref), TINY[dt])
    err = np.abs(out.double().cpu().numpy() - ref)
    assert np.isfinite(err).all()
    worst = (err - tol).max()
    assert worst <= 0, (worst, err.max(), float((err / np.maximum(tol, 1e-300)).max()))


def attention_case(seed, dt, heads, kv, d, page, pos, new, window=0, spread=0.5, scale=None):
    """pos: tokens held per sequence; new: new rows per sequence (an int, or a list for ragged rows)."""
    rng = np.random.default_rng(seed)
    ragged = not isinstance(new, int)
    counts = new if ragged else [new] * len(pos)
    need = [max(0, -(-(p + t) // page)) for p, t in zip(pos, counts)]
    pages = sum(need) + 2
    pool = host_pool(rng, pages, kv, page, d, spread)
    table = tables(rng, need, pages, junk=pages - 1)
    starts = np.concatenate([[0], np.cumsum(counts)])
    n = int(starts[-1])
    q = torch.from_numpy(rng.standard_normal((n, heads, d)).astype(np.float32)).to(TYPES[dt])
    K.device_status(reset=True)
    out = lb.kv8_attention(q.cuda(), device_pool(pool), i32(table), i32(pos), starts=i32(starts) if ragged else None,
                           max_tokens=max(counts) if ragged else None, window=window, scale=scale)
    assert out.dtype == TYPES[dt] and out.shape == (n, heads, d)
    ref, mag, size = R.attention(pool, q.double().numpy(), table, pos, starts, window, scale)
    check(out, ref, mag, size, dt, d, max(p + t for p, t in zip(pos, counts)))
    assert K.device_status(reset=True) == 0


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("heads,kv,d,page", [(4, 2, 32, 16), (14, 2, 64, 64), (8, 8, 64, 32), (32, 8, 128, 128),
                                             (16, 1, 128, 16), (40, 2, 64, 64), (3, 1, 32, 128)])
def test_one_token(dt, heads, kv, d, page):
    pos = [-1, 0, 1, page - 2, page - 1, page, 3 * page + 5, 333]
    attention_case(1, dt, heads, kv, d, page, pos, 1)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("heads,kv,d,page", [(14, 2, 64, 64), (32, 8, 128, 16), (16, 1, 32, 32)])
@pytest.mark.parametrize("new", [2, 5, [0, 1, 7, 3]])
def test_few_tokens(dt, heads, kv, d, page, new):
    attention_case(2, dt, heads, kv, d, page, [0, 3, 200, -2], new)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("heads,kv,d,page", [(14, 2, 64, 64), (8, 2, 128, 64), (4, 4, 32, 16), (6, 1, 64, 128),
                                             (16, 1, 128, 32)])
@pytest.mark.parametrize("new", [33, [130, 1, 0, 61], [257, 128, 64, 300]])
def test_prompts(dt, heads, kv, d, page, new):
    attention_case(3, dt, heads, kv, d, page, [0, 70, 1, -5], new)


def kernels_of(call):
    """Names of the kernels a call launches."""
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA], acc_events=True) as prof:
        call()
        torch.cuda.synchronize()
    return " ".join(e.name for e in prof.events())


def test_many_rows_take_the_prompt_kernel():
    """Few rows stay on the few-row kernel, whatever the lengths; a batch of prompts goes to the other one."""
    cache = lb.KV8Cache.empty(64, 4, 64, page=32)
    for b, new, want, other in ((12, 1, "attention_kernel", "prompt_kernel"), (1, 100, "attention_kernel", "prompt_kernel"),
                                (12, 100, "prompt_kernel", "attention_kernel")):
        q, table, pos = torch.zeros((b * new, 8, 64), device="cuda"), i32(np.zeros((b, 8))), i32([0] * b)
        lb.kv8_attention(q, cache, table, pos)
        names = kernels_of(lambda: lb.kv8_attention(q, cache, table, pos))  # noqa: B023
        assert want in names and other not in names, names


# twelve sequences, so that the calls reach the prompt kernel
LONG = dict(pos=[0, 70, 1, -5, 200, 31, 0, 64, 127, 128, 300, 5], new=[150, 1, 0, 61, 149, 64, 150, 150, 33, 128, 90, 150])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("heads,kv,d,page", [(8, 4, 32, 16), (8, 4, 64, 32), (8, 4, 128, 64), (12, 3, 32, 128), (7, 1, 128, 16),
                                             (30, 2, 64, 128)])
def test_batches_of_prompts(dt, heads, kv, d, page):
    attention_case(13, dt, heads, kv, d, page, **LONG)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("d,page", [(32, 32), (64, 16), (128, 128)])
@pytest.mark.parametrize("window", [1, 40, 64, 129, 1000])
def test_batches_of_prompts_with_windows(dt, d, page, window):
    attention_case(14, dt, 8, 4, d, page, window=window, **LONG)


@pytest.mark.parametrize("dt", TYPES)
def test_batches_of_prompts_long(dt):
    attention_case(15, dt, 8, 4, 64, 64, [1500] * 10 + [0, 1300], 70)


@pytest.mark.parametrize("dt", TYPES)
def test_batches_of_prompts_nothing_leaks(dt):
    """As test_nothing_leaks_from_masked_places, on the prompt kernel."""
    rng = np.random.default_rng(16)
    b, new, window, page, p0 = 12, 100, 40, 16, 110
    width = -(-(p0 + new) // page) + 2
    pool = host_pool(rng, b * width, 4, page, 64)
    table = rng.permutation(b * width).reshape(b, width)
    first = (p0 - window + 1) // page
    q = torch.from_numpy(rng.standard_normal((b * new, 8, 64)).astype(np.float32)).to(TYPES[dt])
    ref, mag, size = R.attention(pool, q.double().numpy(), table, [p0] * b, window=window)
    bad = {n: a.copy() for n, a in pool.items()}
    for n in ("k_exp", "v_exp"):
        bad[n][table[:, :first]] = 255
        bad[n][table[:, -2:]] = 255
    junk = table.copy()
    junk[:, :first], junk[:, -2:] = 10 ** 6, -3
    K.device_status(reset=True)
    for t in (table, junk):
        out = lb.kv8_attention(q.cuda(), device_pool(bad), i32(t), i32([p0] * b), window=window)
        check(out, ref, mag, size, dt, 64, p0 + new)
    assert K.device_status(reset=True) == 0
    o, row = p0 // page + 2, 3  # a NaN block inside sequence 3: exactly the rows that see it
    for n in ("k_exp", "v_exp"):
        one = {m: a.copy() for m, a in bad.items()}
        one[n][table[row, o], 1] = 255
        out = lb.kv8_attention(q.cuda(), device_pool(one), i32(table), i32([p0] * b), window=window).float().cpu().numpy()
        p = np.arange(p0, p0 + new)
        sees = np.zeros((b, new, 8), bool)
        sees[row, :, 2:4] = ((p >= o * page) & (p - window + 1 < (o + 1) * page))[:, None]
        sees = sees.reshape(b * new, 8)
        assert np.isnan(out[sees]).all() and np.isfinite(out[~sees]).all()
    q[5 * new + 1, 2], q[7 * new, 0, 5] = float("nan"), float("inf")
    out = lb.kv8_attention(q.cuda(), device_pool(bad), i32(table), i32([p0] * b), window=window).float().cpu().numpy()
    hit = np.zeros((b * new, 8), bool)
    hit[5 * new + 1, 2] = hit[7 * new, 0] = True
    assert np.isnan(out[hit]).any(-1).all() and np.isfinite(out[~hit]).all()


def test_batches_of_prompts_out_of_range():
    rng = np.random.default_rng(17)
    b, new = 12, 100
    pool = host_pool(rng, 4 * b, 4, 64, 64)
    cache, q = device_pool(pool), torch.randn((b * new, 8, 64), device="cuda")
    table = i32(np.arange(4 * b).reshape(b, 4))
    K.device_status(reset=True)
    good = lb.kv8_attention(q, cache, table, i32([100] * b))
    assert K.device_status(reset=True) == 0
    bad = table.clone()
    bad[0, 0], bad[0, 1] = 4 * b, -1
    out = lb.kv8_attention(q, cache, bad, i32([100] * b))
    assert K.device_status(reset=True) == ERR_PAGE
    assert torch.equal(out[new:], good[new:]) and torch.isfinite(out).all()
    out = lb.kv8_attention(q, cache, table, i32([2 ** 31 - 200] + [100] * (b - 1)))
    assert K.device_status(reset=True) == ERR_PAGE
    assert torch.equal(out[new:], good[new:]) and not out[:new].any()
    st = i32(np.arange(b + 1) * new)
    out = lb.kv8_attention(q, cache, table, i32([100] * b), starts=st, max_tokens=new - 1, out=torch.full_like(good, 7.0))
    assert K.device_status(reset=True) == ERR_PAGE
    ref, mag, size = (a.reshape(b, new, *a.shape[1:])[:, :-1]
                      for a in R.attention(pool, q.cpu().numpy(), table.cpu().numpy(), [100] * b))
    out = out.view(b, new, 8, 64)
    check(out[:, :-1], ref, mag, size, "fp32", 64, 200)
    assert (out[:, -1] == 7).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("b,new", [(1, 1), (9, 1), (3, 40), (12, 150)])
def test_same_bits_every_time(dt, b, new):
    """No result depends on the order in which blocks run; calls on two streams do not disturb each other."""
    rng = np.random.default_rng(18)
    pool = device_pool(host_pool(rng, 20 * b, 4, 64, 64))
    table, pos = i32(rng.permutation(20 * b).reshape(b, 20)), i32([1280 - new - 13 * i for i in range(b)])
    q = torch.randn((b * new, 8, 64), device="cuda").to(TYPES[dt])
    first = lb.kv8_attention(q, pool, table, pos)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(lb.kv8_attention(q, pool, table, pos))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, first)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("window", [1, 2, 15, 64, 100, 5000])
@pytest.mark.parametrize("new", [1, 4, 150])
def test_windows(dt, window, new):
    attention_case(4, dt, 8, 2, 64, 32, [0, 31, 64, 217], new, window=window)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("new,pos", [(1, [4999]), (1, [2600, 17]), (3, [1500]), (200, [1900])])
def test_long(dt, new, pos):
    attention_case(5, dt, 14, 2, 64, 64, pos, new)
    attention_case(6, dt, 4, 1, 128, 16, pos, new)


@pytest.mark.parametrize("new", [1, 2, 40])
@pytest.mark.parametrize("kv,g,d", [(8, 1, 128), (8, 4, 64), (4, 16, 32)])
def test_long_sums_do_not_drift(new, kv, g, d):
    """Positive values, so that sums cut off instead of rounded would all come out small. Rounding to nearest
    has mean 0; what tensor cores cut off stays within a step: two additions to its sum (2 * 2^-23), and as
    much again for the weights' two pieces. So the mean relative error is at most 2^-21."""
    rng = np.random.default_rng(30)
    b, length, page = 64, 8192, 64
    pool = host_pool(rng, length // page, kv, page, d)
    pool["v"] = np.abs(pool["v"])
    table = np.broadcast_to(np.arange(length // page), (b, length // page))  # one prefix for all
    q = torch.from_numpy(rng.standard_normal((b * new, kv * g, d)).astype(np.float32)).cuda()
    out = lb.kv8_attention(q, device_pool(pool), i32(table), i32([length - new] * b))
    k, v = (torch.from_numpy((pool[n] * R.pow2(pool[n + "_exp"])[..., None, None]).transpose(1, 0, 2, 3).reshape(kv, length, d)).cuda()
            for n in "kv")
    worst = []
    for i in range(0, b * new, 8 * new):
        x = q[i:i + 8 * new].double().view(8, new, kv, g, d)
        s = torch.einsum("btkgd,kld->btkgl", x, k) / d ** 0.5
        seen = torch.arange(length, device="cuda") <= torch.arange(length - new, length, device="cuda")[:, None]
        ref = torch.einsum("btkgl,kld->btkgd", s.masked_fill(~seen[None, :, None, None], -torch.inf).softmax(-1), v)
        worst.append(((out[i:i + 8 * new].double().view_as(ref) - ref) / ref).mean().item())
    assert abs(np.mean(worst)) <= 2.0 ** -21, np.mean(worst)


@pytest.mark.parametrize("new", [1, 140])
def test_block_scales_far_apart(new):
    """Blocks 2^20 apart in scale, and an all-zero block (exponent 0) whose tokens still count."""
    rng = np.random.default_rng(7)
    pool = host_pool(rng, 12, 2, 16, 64, 0.0)
    pool["v_exp"] = (pool["v_exp"] + rng.integers(-20, 1, pool["v_exp"].shape)).astype(np.uint8)
    table = rng.permutation(12)[None]
    for n in ("v", "v_exp"):
        pool[n][table[0, 3]] = 0
    pool["k_exp"][table[0, 5]] -= 20
    pos = [180 - new]
    q = rng.standard_normal((new, 4, 64)).astype(np.float32)
    out = lb.kv8_attention(torch.from_numpy(q).cuda(), device_pool(pool), i32(table), i32(pos))
    ref, mag, size = R.attention(pool, q, table, pos)
    check(out, ref, mag, size, "fp32", 64, 180)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("new", [1, 130])
def test_query_magnitudes(dt, new):
    """Queries of very different size, zero ones, and a scale of the caller's."""
    rng = np.random.default_rng(8)
    pool = host_pool(rng, 6, 2, 64, 64)
    table = rng.permutation(6)[None]
    f = np.array([1e-4, 1.0, 5e3, 0.0])[rng.integers(0, 4, (new, 4))][..., None]
    q = torch.from_numpy((rng.standard_normal((new, 4, 64)) * f).astype(np.float32)).to(TYPES[dt])
    for scale in (1e-4, 1e-5):
        out = lb.kv8_attention(q.cuda(), device_pool(pool), i32(table), i32([384 - new]), scale=scale)
        ref, mag, size = R.attention(pool, q.double().numpy(), table, [384 - new], scale=scale)
        check(out, ref, mag, size, dt, 64, 384)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("new", [1, 6, 150])
def test_nothing_leaks_from_masked_places(dt, new):
    """NaN blocks past the sequence and before the window, junk ids there: the rows that do not see them are
    those of a clean pool. A NaN or infinite query spoils its own row only."""
    rng = np.random.default_rng(9)
    pool = host_pool(rng, 16, 2, 16, 64)
    table = rng.permutation(16)[None].copy()
    p0, window = 210 - new, 40
    first = max(0, p0 - window + 1) // 16  # pages before it are seen by no row
    q = torch.from_numpy(rng.standard_normal((new, 4, 64)).astype(np.float32)).to(TYPES[dt])
    ref, mag, size = R.attention(pool, q.double().numpy(), table, [p0], window=window)
    bad = {n: a.copy() for n, a in pool.items()}
    for o in list(range(first)) + [14, 15]:
        for n in ("k_exp", "v_exp"):
            bad[n][table[0, o]] = 255
    out = lb.kv8_attention(q.cuda(), device_pool(bad), i32(table), i32([p0]), window=window)
    check(out, ref, mag, size, dt, 64, 210)
    table[0, :first] = 99999
    table[0, 14:] = -7
    out = lb.kv8_attention(q.cuda(), device_pool(bad), i32(table), i32([p0]), window=window)
    check(out, ref, mag, size, dt, 64, 210)
    assert K.device_status(reset=True) == 0
    if new > 1:
        # a NaN block inside: exactly the rows that see it
        o = (p0 + new - 1 - window - 2) // 16 if new > 60 else p0 // 16 - 1
        for n in ("k_exp", "v_exp"):
            one = {m: a.copy() for m, a in bad.items()}
            one[n][table[0, o], 1] = 255
            out = lb.kv8_attention(q.cuda(), device_pool(one), i32(table), i32([p0]), window=window).float().cpu().numpy()
            p = np.arange(p0, p0 + new)
            sees = (p >= o * 16) & (p - window + 1 < (o + 1) * 16)
            assert np.isnan(out[sees][:, 2:]).all()
            assert np.isfinite(out[:, :2]).all() and np.isfinite(out[~sees]).all()
        q[1, 2] = float("nan")
        q[0, 0, 5] = float("inf")
        out = lb.kv8_attention(q.cuda(), device_pool(bad), i32(table), i32([p0]), window=window).float().cpu().numpy()
        hit = np.zeros((new, 4), bool)
        hit[1, 2] = hit[0, 0] = True
        assert np.isnan(out[hit]).any(-1).all() and np.isfinite(out[~hit]).all()


@pytest.mark.parametrize("new", [1, 140])
def test_out_of_range_is_recorded_and_skipped(new):
    rng = np.random.default_rng(10)
    pool = host_pool(rng, 8, 2, 64, 64)
    cache, q = device_pool(pool), torch.randn((2 * new, 4, 64), device="cuda")
    table = i32([[0, 1, 2, 3], [4, 5, 6, 7]])
    K.device_status(reset=True)
    good = lb.kv8_attention(q, cache, table, i32([100, 100]))
    assert K.device_status(reset=True) == 0
    bad = table.clone()
    bad[0, 0], bad[0, 1] = 8, -1
    out = lb.kv8_attention(q, cache, bad, i32([100, 100]))
    assert K.device_status(reset=True) == ERR_PAGE
    assert torch.equal(out[new:], good[new:])
    out = lb.kv8_attention(q, cache, table, i32([2 ** 31 - 200, 100]))  # past the table: nothing to see
    assert K.device_status(reset=True) == ERR_PAGE
    assert torch.equal(out[new:], good[new:]) and not out[:new].any()
    if new > 1:  # more rows than max_tokens: the first max_tokens are computed
        st = i32([0, new, 2 * new])
        out = lb.kv8_attention(q, cache, table, i32([100, 100]), starts=st, max_tokens=new - 1,
                               out=torch.full_like(good, 7.0))
        assert K.device_status(reset=True) == ERR_PAGE
        assert torch.isfinite(out[:new - 1]).all() and torch.equal(out[new - 1], torch.full_like(out[0], 7.0))


@pytest.mark.parametrize("dt", TYPES)
def test_batches_of_prompts_strided(dt):
    """q as a slice of fused rows, on the prompt kernel: the same bits."""
    rng = np.random.default_rng(19)
    cache = device_pool(host_pool(rng, 48, 4, 64, 64))
    table, pos = i32(rng.permutation(48).reshape(12, 4)), i32([100] * 12)
    q = torch.randn((1200, 16 * 64), device="cuda").to(TYPES[dt])[:, 256:768].unflatten(1, (8, 64))
    assert not q.is_contiguous()
    assert torch.equal(lb.kv8_attention(q, cache, table, pos), lb.kv8_attention(q.contiguous(), cache, table, pos))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("new", [1, 3, 140])
def test_strides(dt, new):
    """q as a slice of fused rows, misaligned q, pages with gaps: the same bits as dense tensors."""
    rng = np.random.default_rng(11)
    pool = host_pool(rng, 9, 2, 32, 64)
    table, pos = i32(rng.permutation(9)[None]), i32([270 - new])
    rows = torch.randn((new, 8 * 64), device="cuda").to(TYPES[dt])
    q = rows[:, 64:5 * 64].unflatten(1, (4, 64))
    ref = lb.kv8_attention(q.contiguous(), device_pool(pool), table, pos)
    assert torch.equal(lb.kv8_attention(q, device_pool(pool), table, pos), ref)
    flat = torch.zeros(q.numel() + 1, dtype=q.dtype, device="cuda")
    flat[1:] = q.reshape(-1)
    assert torch.equal(lb.kv8_attention(flat[1:].view(new, 4, 64), device_pool(pool), table, pos), ref)
    assert torch.equal(lb.kv8_attention(q.transpose(1, 2).contiguous().transpose(1, 2), device_pool(pool), table, pos), ref)
    both = torch.zeros((9, 2, 2, 32, 64), dtype=torch.int8, device="cuda")
    exps = torch.zeros((9, 2, 3), dtype=torch.uint8, device="cuda")
    c = device_pool(pool)
    both[:, 0], both[:, 1], exps[:, 0, :2], exps[:, 1, 1:] = c.k, c.v, c.k_exp, c.v_exp
    wide = lb.KV8Cache(both[:, 0], both[:, 1], exps[:, 0, :2], exps[:, 1, 1:])
    assert torch.equal(lb.kv8_attention(q, wide, table, pos), ref)
    for a, b in zip(lb.kv8_read(wide, table[0]), lb.kv8_read(c, table[0])):
        assert torch.equal(a, b)


@pytest.mark.parametrize("new", [1, 140])
def test_pools_past_32_bit_offsets(new):
    """Pages 1.5 GiB apart: the last one starts past 2^32 bytes."""
    rng = np.random.default_rng(12)
    pool = host_pool(rng, 4, 1, 64, 64)
    gap = 3 << 29
    raw = torch.empty(3 * gap + 64 * 64 * 2, dtype=torch.int8, device="cuda")
    k = raw.as_strided((4, 1, 64, 64), (gap, 4096, 64, 1))
    v = raw.as_strided((4, 1, 64, 64), (gap, 4096, 64, 1), 4096)
    dense = device_pool(pool)
    k.copy_(dense.k)
    v.copy_(dense.v)
    far = lb.KV8Cache(k, v, dense.k_exp.clone(), dense.v_exp.clone())
    table, pos = i32([[3, 0, 2, 1]]), i32([256 - new])
    q = torch.randn((new, 2, 64), device="cuda")
    assert torch.equal(lb.kv8_attention(q, far, table, pos), lb.kv8_attention(q, dense, table, pos))
    cos, sin = (torch.from_numpy(t).cuda() for t in rope_tables(64, 256, 1e4))
    qkv = torch.randn((new, 4 * 64), device="cuda")
    assert torch.equal(lb.kv8_append(qkv, far, table, pos, cos, sin), lb.kv8_append(qkv, dense, table, pos, cos, sin))
    for a, b in zip(lb.kv8_read(far, table[0]), lb.kv8_read(dense, table[0])):
        assert torch.equal(a, b)


# ---------------------------------------------------------------- append and read

def same_pool(cache, pool):
    for n in ("k", "v", "k_exp", "v_exp"):
        np.testing.assert_array_equal(getattr(cache, n).cpu().numpy(), pool[n])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("heads,kv,d,page", [(4, 2, 32, 16), (14, 2, 64, 64), (8, 8, 64, 32), (8, 2, 128, 128), (16, 1, 128, 16)])
@pytest.mark.parametrize("new", [1, 3, [0, 1, 70, 5], [129, 128, 1, 257]])
def test_append(dt, heads, kv, d, page, new):
    rng = np.random.default_rng(20)
    pos = [0, page - 1, 2 * page + 3, -2]
    counts = [new] * 4 if isinstance(new, int) else new
    need = [max(0, -(-(p + t) // page)) for p, t in zip(pos, counts)]
    pool = host_pool(rng, sum(need) + 1, kv, page, d)
    table = tables(rng, need, sum(need) + 1, junk=-1)
    starts = np.concatenate([[0], np.cumsum(counts)])
    n, w = int(starts[-1]), (heads + 2 * kv) * d
    # magnitudes from row to row, so that some blocks grow and others do not
    x = rng.standard_normal((n, w)) * np.exp(rng.standard_normal((n, 1)))
    qkv = torch.from_numpy(x.astype(np.float32)).to(TYPES[dt])
    cos, sin = rope_tables(d, 3 * page + 300, 1e4)
    bias = rng.standard_normal(w).astype(np.float32) if heads == 14 else None
    cache = device_pool(pool)
    K.device_status(reset=True)
    q = lb.kv8_append(qkv.cuda(), cache, i32(table), i32(pos), torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda(),
                      bias=None if bias is None else torch.from_numpy(bias).cuda(),
                      starts=None if isinstance(new, int) else i32(starts), max_tokens=max(counts))
    ref = R.append(pool, qkv.float().numpy(), table, pos, cos, sin, heads, bias, starts)
    assert torch.equal(q.cpu(), torch.from_numpy(ref).to(TYPES[dt]))
    same_pool(cache, pool)
    assert K.device_status(reset=True) == 0


def test_append_grows_a_block_step_by_step():
    """Token by token into one page, magnitudes rising over 2^40 and falling: every growth shifts the older codes."""
    rng = np.random.default_rng(21)
    pool = host_pool(rng, 1, 1, 32, 32)
    cache, table = device_pool(pool), np.zeros((1, 1), np.int64)
    cos, sin = rope_tables(32, 32, 1e4)
    for t in range(32):
        x = (rng.standard_normal((1, 4 * 32)) * 2.0 ** (2 * min(t, 40 - t) - 20)).astype(np.float32)
        if t == 3:
            x[:] = 0
        q = lb.kv8_append(torch.from_numpy(x).cuda(), cache, i32(table), i32([t]), torch.from_numpy(cos).cuda(),
                          torch.from_numpy(sin).cuda())
        np.testing.assert_array_equal(q.cpu().numpy(), R.append(pool, x, table, [t], cos, sin, 2))
        same_pool(cache, pool)


def test_append_non_finite_and_extreme_values():
    rng = np.random.default_rng(22)
    pool = host_pool(rng, 4, 2, 16, 32)
    cache, table = device_pool(pool), np.array([[3, 1, 0, 2]])
    cos, sin = rope_tables(32, 64, 1e4)
    cos, sin = np.ones_like(cos), np.zeros_like(sin)
    x = rng.standard_normal((64, 6 * 32)).astype(np.float32)
    top = np.finfo(np.float32).max
    x[2, 2 * 32] = np.nan             # k of head 0, page 0
    x[20, 4 * 32 + 1] = np.inf        # v of head 0, page 1
    x[33, 3 * 32:4 * 32] = top        # k of head 1, page 2
    x[48:, 5 * 32:] = 1e-42           # v of head 1, page 3: subnormal
    x[48:, 3 * 32:4 * 32] = 0
    with np.errstate(over="ignore", invalid="ignore"):
        ref = R.append(pool, x, table, [0], cos, sin, 2)
    q = lb.kv8_append(torch.from_numpy(x).cuda(), cache, i32(table), i32([0]), torch.from_numpy(cos).cuda(),
                      torch.from_numpy(sin).cuda())
    np.testing.assert_array_equal(q.cpu().numpy(), ref)
    same_pool(cache, pool)
    assert pool["k_exp"][3, 0] == 255 and pool["v_exp"][1, 0] == 255 and pool["v_exp"][2, 1] == 0
    k, v = lb.kv8_read(cache, i32(table[0]), dtype=torch.float32)
    assert torch.isnan(k[0, 0]).all() and torch.isnan(v[1, 0]).all() and torch.isfinite(k[1:]).all()
    # a NaN block stays one until it is begun anew
    y = torch.ones((1, 6 * 32), device="cuda")
    c, s = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
    lb.kv8_append(y, cache, i32(table), i32([5]), c, s)
    assert int(cache.k_exp[3, 0]) == 255
    lb.kv8_append(y, cache, i32(table), i32([0]), c, s)
    assert int(cache.k_exp[3, 0]) == 121


def test_append_out_of_range_is_recorded_and_skipped():
    rng = np.random.default_rng(23)
    pool = host_pool(rng, 4, 2, 16, 32)
    cos, sin = rope_tables(32, 40, 1e4)
    c, s = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
    x = rng.standard_normal((30, 6 * 32)).astype(np.float32)
    K.device_status(reset=True)
    for table, pos in (([[0, 9, 2]], 0), ([[0, -1, 2]], 8), ([[0, 1]], 5), ([[0, 1, 2]], 15), ([[0, 1, 2]], 2 ** 31 - 4)):
        p = {n: a.copy() for n, a in pool.items()}
        cache = device_pool(p)
        q = lb.kv8_append(torch.from_numpy(x).cuda(), cache, i32(table), i32([pos]), c, s)
        assert K.device_status(reset=True) == ERR_PAGE
        ref = R.append(p, x, np.array(table), [pos], cos, sin, 2)
        np.testing.assert_array_equal(q.cpu().numpy(), ref)
        same_pool(cache, p)
    cache = device_pool(pool)
    k, v = lb.kv8_read(cache, i32([1, 4, -1]))
    assert K.device_status(reset=True) == ERR_PAGE
    assert k[0].any() and not k[1:].any() and not v[1:].any()


@pytest.mark.parametrize("d,page,kv", [(32, 16, 1), (64, 64, 2), (128, 128, 3)])
def test_read(d, page, kv):
    rng = np.random.default_rng(24)
    pool = host_pool(rng, 7, kv, page, d)
    pool["k_exp"][3, 0], pool["v_exp"][2, 0], pool["v_exp"][1, 0] = 0, 255, 249
    cache, ids = device_pool(pool), [3, 0, 2, 2, 1]
    for dt in TYPES.values():
        got = lb.kv8_read(cache, i32(ids), dtype=dt)
        for n, g in zip("kv", got):
            ref = pool[n][ids] * R.pow2(pool[n + "_exp"][ids])[..., None, None]
            assert g.dtype == dt
            assert torch.equal(g.cpu().nan_to_num(1.25), torch.from_numpy(ref).float().to(dt).nan_to_num(1.25))
    assert [t.shape[0] for t in lb.kv8_read(cache, i32([]))] == [0, 0]


@pytest.mark.parametrize("d,page,kv,n", [(32, 16, 3, 701), (64, 16, 5, 333), (32, 64, 1, 1500), (128, 64, 3, 450)])
def test_read_many_blocks(d, page, kv, n):
    rng = np.random.default_rng(25)
    pool = host_pool(rng, 9, kv, page, d)
    pool["v_exp"][4, 0] = 255
    cache, ids = device_pool(pool), rng.integers(0, 9, n)
    bad = ids.copy()
    bad[[0, n // 2, n - 1]] = [9, -1, 2 ** 31 - 1]
    K.device_status(reset=True)
    for dt in TYPES.values():
        for want in (ids, bad):
            got = lb.kv8_read(cache, i32(want), dtype=dt)
            there = (want >= 0) & (want < 9)
            for name, g in zip("kv", got):
                ref = pool[name][want * there] * R.pow2(pool[name + "_exp"][want * there])[..., None, None]
                ref[~there] = 0
                assert torch.equal(g.cpu().nan_to_num(1.25), torch.from_numpy(ref).float().to(dt).nan_to_num(1.25))
            assert K.device_status(reset=True) == (0 if there.all() else ERR_PAGE)


# ---------------------------------------------------------------- streams, graphs, refusals

def test_another_stream_and_graph_replay():
    """Append and attention captured once, replayed with new rows, positions and tables."""
    rng = np.random.default_rng(30)
    pool = host_pool(rng, 24, 2, 16, 64)
    cos, sin = rope_tables(64, 200, 1e4)
    c, s = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
    cache = device_pool(pool)
    table, pos = i32(np.zeros((2, 12))), i32([-1, -1])
    qkv = torch.zeros((2, 8 * 64), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lb.kv8_attention(lb.kv8_append(qkv, cache, table, pos, c, s), cache, table, pos)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q = lb.kv8_append(qkv, cache, table, pos, c, s)
        out = lb.kv8_attention(q, cache, table, pos)
    ids = rng.permutation(24).reshape(2, 12)
    for step, p in enumerate([[0, 100], [1, 101], [2, -1], [150, 191]]):
        x = rng.standard_normal((2, 8 * 64)).astype(np.float32)
        t = ids if step % 2 == 0 else ids[::-1].copy()
        qkv.copy_(torch.from_numpy(x))
        table.copy_(i32(t))
        pos.copy_(i32(p))
        g.replay()
        qr = R.append(pool, x, t, p, cos, sin, 4)
        np.testing.assert_array_equal(q.cpu().numpy(), qr)
        same_pool(cache, pool)
        check(out, *R.attention(pool, qr, t, p), "fp32", 64, 192)


def test_refusals():
    cache = lb.KV8Cache.empty(4, 2, 64, page=32)
    assert cache.nbytes == 2 * 4 * 2 * (32 * 64 + 1)
    q, table, pos = torch.zeros((2, 4, 64), device="cuda"), i32([[0, 1], [2, 3]]), i32([0, 0])
    ok = lb.kv8_attention(q, cache, table, pos)
    assert not ok.any()
    for kw in (dict(q=q.double()), dict(q=q.cpu()), dict(q=q[:, :3]), dict(q=q[:, :, :32]), dict(q=q[0]), dict(table=table.long()),
               dict(table=table.cpu()), dict(table=table[:, :0]), dict(pos=pos[:1]), dict(pos=pos.float()), dict(window=-1),
               dict(starts=i32([0, 2])), dict(q=q[:1]), dict(max_tokens=0), dict(starts=i32([0, 1, 2]), max_tokens=-1),
               dict(out=ok[:1]), dict(out=ok.half())):
        args = dict(q=q, cache=cache, table=table, pos=pos) | kw
        with pytest.raises(ValueError):
            lb.kv8_attention(**args)
    cos, sin = (torch.from_numpy(t).cuda() for t in rope_tables(64, 64, 1e4))
    qkv = torch.zeros((2, 8 * 64), device="cuda")
    for kw in (dict(qkv=qkv[:, :4 * 64]), dict(qkv=qkv[:, :500]), dict(qkv=qkv.int()), dict(cos=cos[:, :16]), dict(sin=sin[:32]),
               dict(cos=cos.double()), dict(bias=torch.zeros(5, device="cuda")), dict(bias=torch.zeros(512)), dict(pos=pos.cpu())):
        args = dict(qkv=qkv, cache=cache, table=table, pos=pos, cos=cos, sin=sin) | kw
        with pytest.raises(ValueError):
            lb.kv8_append(**args)
    for pages, dt in ((i32([[0]]), torch.float32), (i32([0]).long(), torch.float32), (i32([0]), torch.float64)):
        with pytest.raises(ValueError):
            lb.kv8_read(cache, pages, dtype=dt)
    k, e = cache.k, cache.k_exp
    for bad in ((k[:, :, :24], k[:, :, :24], e, e), (k.transpose(0, 1), k.transpose(0, 1), e.T, e.T), (k, k[:2], e, e),
                (k, k, e[:2], e), (k[:, :1].expand(4, 2, 32, 64), k, e, e)):
        with pytest.raises(ValueError):
            lb.KV8Cache(*bad)
    assert lb.kv8_attention(q[:0], cache, table, pos).shape == (0, 4, 64)
