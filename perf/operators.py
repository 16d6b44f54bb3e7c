"""Measured cases of the 8-bit paged KV-cache operators, with their plain forms.

The cache is a pool of pages: int8 codes [pages, KV, P, D] for keys and for
values and one power-of-two scale byte per page and head (E8M0: a code stands
for code * 2^(e - 127)). Three operators work on it:

* append     bias and rotate-half position rotation of fused q/k/v rows, k and
             v quantised into the pages of their sequences, q rotated;
* attention  causal grouped-query attention of new tokens over the pages, with
             an optional sliding window;
* read       pages back as values.

`run` computes a case either in plain torch operations (`own` false) or with
the framework's entry points (`own` true).
"""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------- cases

def listed():
    """Head layouts: 14 query and 2 KV heads of 64 (the framework's Qwen2-0.5B
    shape, fp32 with qkv bias) and a generic 32 / 8 heads of 128. `past` is the
    longest number of tokens already held, `new` the most tokens a sequence
    brings; `ragged` draws both per sequence from `mix`."""
    small = {"heads": 14, "kv": 2, "dim": 64, "page": 64, "dtype": "fp32", "window": 0}
    large = {"heads": 32, "kv": 8, "dim": 128, "page": 64, "dtype": "bf16", "window": 0}
    return [
        # one user, one token: the latency of a decode step
        {"name": "append_one", "op": "append", **small, "batch": 1, "new": 1, "past": 509, "ragged": False, "mix": 1},
        # a serving batch's decode step, sequences of very different lengths
        {"name": "append_decode_64", "op": "append", **large, "batch": 64, "new": 1, "past": 4000, "ragged": True, "mix": 2},
        # prompts of different lengths joining part-filled sequences
        {"name": "append_prompts", "op": "append", **large, "batch": 5, "new": 2047, "past": 300, "ragged": True, "mix": 3},
        # one user, one token, a short chat
        {"name": "decode_one", "op": "attention", **small, "batch": 1, "new": 1, "past": 509, "ragged": False, "mix": 4},
        # the batch-16 decode of the framework's model at its largest context
        {"name": "decode_16", "op": "attention", **small, "batch": 16, "new": 1, "past": 4095, "ragged": True, "mix": 5},
        # a full serving batch
        {"name": "decode_64", "op": "attention", **large, "batch": 64, "new": 1, "past": 8191, "ragged": True, "mix": 6},
        # one user with a long document
        {"name": "decode_long", "op": "attention", **large, "batch": 1, "new": 1, "past": 131070, "ragged": False, "mix": 7},
        # checking five drafted tokens a sequence under a sliding window, small pages, fp16
        {"name": "verify_window", "op": "attention", **large, "dtype": "fp16", "page": 16, "window": 1024, "batch": 16,
         "new": 5, "past": 4000, "ragged": True, "mix": 8},
        # a prompt chunk of the framework's model after an equally long context, fp32
        {"name": "chunk_fp32", "op": "attention", **small, "batch": 1, "new": 2048, "past": 2047, "ragged": False, "mix": 9},
        # whole prompts of different lengths
        {"name": "prompts", "op": "attention", **large, "batch": 2, "new": 4096, "past": 0, "ragged": True, "mix": 10},
        # a short prefix handed to another engine, and a long one
        {"name": "read_prefix", "op": "read", **small, "batch": 1, "new": 0, "past": 509, "ragged": False, "mix": 11},
        {"name": "read_document", "op": "read", **large, "batch": 1, "new": 0, "past": 65536, "ragged": False, "mix": 12},
    ]


def draw(rng):
    """One more case: both head layouts' neighbours, every head size, page size
    and type, lengths spread over their logarithm."""
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        heads, kv = rng.choice([(4, 2), (14, 2), (32, 8), (8, 8), (16, 1), (28, 4)])
        op = rng.choice(["append", "attention", "attention", "attention", "read"])
        form = "read" if op == "read" else rng.choice(["one", "one", "few", "prompt"])
        case = {"op": op, "heads": heads, "kv": kv, "dim": rng.choice([32, 64, 128]), "page": rng.choice([16, 32, 64, 128]),
                "dtype": rng.choice(["fp32", "bf16", "bf16", "fp16"]), "window": 0, "batch": spread(1, 64),
                "past": spread(1, 65536) - 1, "ragged": rng.random() < 0.7, "mix": rng.randrange(1, 1 << 30)}
        case["new"] = {"read": 0, "one": 1, "few": rng.randrange(2, 10), "prompt": spread(10, 4096)}[form]
        if op == "attention" and rng.random() < 0.25:
            case["window"] = spread(16, 4096)
        if op == "read":
            case["past"] = max(1, case["past"])
        if form == "prompt":
            case["batch"], case["past"] = min(case["batch"], 4), min(case["past"], 8192)
        w, pool = work(case), case["batch"] * (case["past"] + case["new"]) * kv * case["dim"] * 2
        dense = case["batch"] * heads * case["new"] * (case["past"] + case["new"])
        if w["bytes"] <= 8e8 and w["flops"] <= 2.6e11 and pool <= 8e8 and dense <= 1.0e9:
            return case


def lengths(case):
    """Tokens held and tokens new, per sequence."""
    rng = random.Random(case["mix"])
    b, past, new = case["batch"], case["past"], case["new"]
    if not case["ragged"]:
        return [past] * b, [new] * b
    held = [rng.randint(past // 8, past) for _ in range(b)]
    held[rng.randrange(b)] = past
    # decode steps bring one token each; longer ones differ from sequence to sequence
    fresh = [new if new <= 1 else rng.randint(max(1, new // 4), new) for _ in range(b)]
    fresh[rng.randrange(b)] = new
    return held, fresh


def work(case):
    held, fresh = lengths(case)
    es = 4 if case["dtype"] == "fp32" else 2
    h, kv, d, page, win = case["heads"], case["kv"], case["dim"], case["page"], case["window"]
    n = sum(fresh)
    if case["op"] == "read":
        pages = sum(-(-p // page) for p in held)
        return {"bytes": 2 * pages * kv * (page * d * 3 + 1), "flops": 2 * pages * kv * page * d}
    if case["op"] == "append":
        pages = sum((p + t - 1) // page - p // page + 1 for p, t in zip(held, fresh))
        # rows in, q out, and the touched pages: codes in and out, values out
        return {"bytes": n * (2 * h + 2 * kv) * d * es + 2 * pages * kv * (page * d * 4 + 2), "flops": 6 * n * (h + 2 * kv) * d}
    keys = pairs = 0
    for p, t in zip(held, fresh):
        first = max(0, p - win + 1) if win else 0
        keys += p + t - first
        if win:
            pairs += sum(min(q + 1, win) for q in range(p, p + t))
        else:
            pairs += t * p + t * (t + 1) // 2
    return {"bytes": 2 * n * h * d * es + 2 * keys * kv * d + 2 * keys * kv // page, "flops": 4 * pairs * h * d}


# ---------------------------------------------------------------- inputs

def pow2(e):
    """2^(e - 127) of E8M0 bytes, from the float's bits."""
    bits = torch.where(e == 0, 0x400000, e.int() << 23).to(torch.int32)
    return bits.view(torch.float32)


def scale_byte(amax):
    """The smallest e >= 0 with amax <= 127 * 2^(e - 127)."""
    m, x = torch.frexp(amax)
    e = torch.where(m > 127 / 128, x - 6, x - 7) + 127
    return torch.where(amax == 0, 0, e.clamp(min=0)).to(torch.uint8)


def pool(pages, kv, page, d, gen):
    """Codes and scale bytes of random keys or values: some channels larger
    than others, pages of different magnitude."""
    x = torch.randn((pages, kv, page, d), generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn((1, kv, 1, d), generator=gen, device="cuda"))
    x *= torch.exp(0.3 * torch.randn((pages, kv, 1, 1), generator=gen, device="cuda"))
    e = scale_byte(x.abs().amax((2, 3)))
    x *= 1.0 / pow2(e)[:, :, None, None]
    return x.round_().to(torch.int8), e


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    held, fresh = lengths(case)
    b, h, kv, d, page = case["batch"], case["heads"], case["kv"], case["dim"], case["page"]
    dtype = DTYPES[case["dtype"]]
    n = sum(fresh)
    per = [-(-(p + t) // page) for p, t in zip(held, fresh)]
    total = sum(per) + 3
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((b, max(per)), dtype=torch.int32)
    at, touched = 0, []
    ids = order.cpu()
    for i, c in enumerate(per):
        table[i, :c] = ids[at:at + c]
        touched.append(ids[at + held[i] // page:at + c])
        at += c
    k, k_exp = pool(total, kv, page, d, gen)
    v, v_exp = pool(total, kv, page, d, gen)
    starts = [0]
    for t in fresh:
        starts.append(starts[-1] + t)
    s = {"op": case["op"], "k": k, "v": v, "k_exp": k_exp, "v_exp": v_exp, "table": table.cuda(),
         "pos": torch.tensor(held, dtype=torch.int32, device="cuda"), "most": max(fresh), "window": case["window"],
         # equal counts need no offsets; a program with ragged rows has them
         "starts": torch.tensor(starts, dtype=torch.int32, device="cuda") if len(set(fresh)) > 1 else None,
         "heads": h}
    if case["op"] == "append":
        s["pages"] = torch.cat(touched).cuda()
        s["qkv"] = (1.3 * torch.randn((n, (h + 2 * kv) * d), generator=gen, device="cuda")).to(dtype)
        # the framework's model has a qkv bias; the generic layout has none
        s["bias"] = 0.3 * torch.randn((h + 2 * kv) * d, generator=gen, device="cuda") if heads_with_bias(case) else None
        inv = 1.0 / 1e6 ** (torch.arange(0, d, 2, dtype=torch.float64) / d)
        ang = torch.arange(case["past"] + case["new"], dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = ang.cos().float().cuda(), ang.sin().float().cuda()
    elif case["op"] == "attention":
        s["q"] = torch.randn((n, h, d), generator=gen, device="cuda").to(dtype)
    else:
        s["pages"] = torch.cat([table[i, :c] for i, c in enumerate(per)]).cuda()
    if own:
        # the handle a program keeps beside its pool (it holds these tensors)
        import lowbit_b200 as lb
        s["cache"] = lb.KV8Cache(k, v, k_exp, v_exp)
    return s


def heads_with_bias(case):
    return case["heads"] == 14


# ---------------------------------------------------------------- one pass

def run(s):
    if own:
        import lowbit_b200 as lb
        if s["op"] == "attention":
            return lb.kv8_attention(s["q"], s["cache"], s["table"], s["pos"], starts=s["starts"], max_tokens=s["most"],
                                    window=s["window"])
        if s["op"] == "read":
            k, v = lb.kv8_read(s["cache"], s["pages"])
            return {"k": k, "v": v}
        q = lb.kv8_append(s["qkv"], s["cache"], s["table"], s["pos"], s["cos"], s["sin"], bias=s["bias"],
                          starts=s["starts"], max_tokens=s["most"])
        k, v = lb.kv8_read(s["cache"], s["pages"])
        return {"q": q, "k": k, "v": v}
    if s["op"] == "attention":
        return plain_attention(s)
    if s["op"] == "read":
        return {"k": plain_read(s["k"], s["k_exp"], s["pages"]), "v": plain_read(s["v"], s["v_exp"], s["pages"])}
    q = plain_append(s)
    return {"q": q, "k": plain_read(s["k"], s["k_exp"], s["pages"]), "v": plain_read(s["v"], s["v_exp"], s["pages"])}


def rows_of(s, n):
    """Sequence, index among its new tokens and position of every row."""
    i = torch.arange(n, device="cuda")
    if s["starts"] is None:
        seq, t = i // s["most"], i % s["most"]
    else:
        seq = torch.searchsorted(s["starts"][1:].long(), i, right=True)
        t = i - s["starts"][seq].long()
    return seq, t, s["pos"][seq].long() + t


def plain_read(codes, e, pages):
    i = pages.long()
    return (codes[i].float() * pow2(e[i])[:, :, None, None]).to(torch.bfloat16)


def plain_store(codes, e, x, page_of, slot):
    """Rows x [N, KV, D] into their blocks: the block's scale grows where the
    new rows need it, and its older codes are rounded to the new step."""
    u, inv = torch.unique(page_of, return_inverse=True)
    fresh = torch.zeros((len(u), codes.shape[2], codes.shape[1], codes.shape[3]), device="cuda")
    fresh[inv, slot] = x
    written = torch.zeros((len(u), codes.shape[2]), dtype=torch.bool, device="cuda")
    written[inv, slot] = True
    older = written.int().cumsum(1) == 0
    old_e = torch.where(written[:, :1], 0, e[u].int())
    new_e = torch.maximum(old_e, scale_byte(fresh.abs().amax((1, 3))).int())
    old = codes[u].float()
    moved = (old * pow2((old_e - new_e + 127).clamp(min=1))[:, :, None, None]).round()
    put = (fresh.permute(0, 2, 1, 3) * (1.0 / pow2(new_e.to(torch.uint8)))[:, :, None, None]).round().clamp(-127, 127)
    older, written = older[:, None, :, None], written[:, None, :, None]
    codes[u] = torch.where(written, put, torch.where(older, moved, old)).to(torch.int8)
    e[u] = new_e.to(torch.uint8)


def plain_append(s):
    qkv, k = s["qkv"], s["k"]
    n, h, kv, d, page = len(qkv), s["heads"], k.shape[1], k.shape[3], k.shape[2]
    seq, _, p = rows_of(s, n)
    x = qkv.float()
    if s["bias"] is not None:
        x = x + s["bias"]
    x = x.view(n, h + 2 * kv, d)
    c, sn = s["cos"][p][:, None], s["sin"][p][:, None]
    x1, x2 = x[:, :h + kv, :d // 2], x[:, :h + kv, d // 2:]
    rot = torch.cat([x1 * c - x2 * sn, x2 * c + x1 * sn], -1)
    page_of = s["table"][seq, p // page].long()
    plain_store(s["k"], s["k_exp"], rot[:, h:], page_of, p % page)
    plain_store(s["v"], s["v_exp"], x[:, h + kv:], page_of, p % page)
    return rot[:, :h].to(qkv.dtype)


def plain_attention(s):
    q, k, v, page = s["q"], s["k"], s["v"], s["k"].shape[2]
    n, h, d = q.shape
    b, kv = len(s["pos"]), k.shape[1]
    t_max, g, size = s["most"], h // kv, s["table"].shape[1] * page
    seq, t, p = rows_of(s, n)
    i = s["table"].long()
    keys = (k[i].float() * pow2(s["k_exp"][i])[..., None, None]).permute(0, 2, 1, 3, 4).reshape(b, kv, size, d)
    vals = (v[i].float() * pow2(s["v_exp"][i])[..., None, None]).permute(0, 2, 1, 3, 4).reshape(b, kv, size, d)
    rows = torch.zeros((b, t_max, h, d), device="cuda")
    rows[seq, t] = q.float()
    rows = rows.view(b, t_max, kv, g, d).permute(0, 2, 3, 1, 4).reshape(b, kv, g * t_max, d)
    score = (rows @ keys.transpose(2, 3)).view(b, kv, g, t_max, size) * (1.0 / math.sqrt(d))
    j = torch.arange(size, device="cuda")
    at = s["pos"].long()[:, None, None] + torch.arange(t_max, device="cuda")[:, None]
    seen = j <= at
    if s["window"]:
        seen = seen & (j > at - s["window"])
    score = torch.where(seen[:, None, None], score, -math.inf)
    score = torch.exp(score - score.amax(-1, keepdim=True))
    score = score / score.sum(-1, keepdim=True)
    out = score.view(b, kv, g * t_max, size) @ vals
    out = out.view(b, kv, g, t_max, d).permute(0, 3, 1, 2, 4).reshape(b, t_max, h, d)
    return out[seq, t].to(q.dtype)


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    """The same outputs from the definitions, in 64 bits, sequence by sequence."""
    s = prepare(case, seed)
    held, fresh = lengths(case)
    page = case["page"]
    f64 = torch.float64

    def values(codes, e, pages):
        return codes[pages].to(f64) * torch.ldexp(torch.ones((), dtype=f64, device="cuda"),
                                                  e[pages].to(f64) - 127)[:, :, None, None]

    if case["op"] == "read":
        i = s["pages"].long()
        return {"k": values(s["k"], s["k_exp"], i), "v": values(s["v"], s["v_exp"], i)}
    if case["op"] == "attention":
        out, row = torch.zeros(s["q"].shape, dtype=f64, device="cuda"), 0
        g, kv, d = case["heads"] // case["kv"], case["kv"], case["dim"]
        for b, (p, t) in enumerate(zip(held, fresh)):
            pages = s["table"][b, :-(-(p + t) // page)].long()
            kk = values(s["k"], s["k_exp"], pages).transpose(0, 1).reshape(kv, -1, d)[:, :p + t]
            vv = values(s["v"], s["v_exp"], pages).transpose(0, 1).reshape(kv, -1, d)[:, :p + t]
            at = torch.arange(p, p + t, device="cuda")[:, None]
            j = torch.arange(p + t, device="cuda")
            hide = j > at
            if case["window"]:
                hide |= j <= at - case["window"]
            for a in range(case["heads"]):
                w = s["q"][row:row + t, a].to(f64) @ kk[a // g].T / math.sqrt(d)
                w = torch.softmax(w.masked_fill(hide, -math.inf), -1)
                out[row:row + t, a] = w @ vv[a // g]
            row += t
        return out
    h, kv, d = case["heads"], case["kv"], case["dim"]
    x = s["qkv"].to(f64)
    if s["bias"] is not None:
        x = x + s["bias"].to(f64)
    x = x.view(-1, h + 2 * kv, d).clone()
    where = torch.cat([torch.arange(p, p + t) for p, t in zip(held, fresh)]).cuda()
    turn = torch.complex(s["cos"].to(f64), s["sin"].to(f64))[where][:, None]
    z = torch.complex(x[:, :h + kv, :d // 2].contiguous(), x[:, :h + kv, d // 2:].contiguous()) * turn
    x[:, :h + kv] = torch.cat([z.real, z.imag], -1)
    both = []
    for codes, e, new in ((s["k"], s["k_exp"], x[:, h:h + kv]), (s["v"], s["v_exp"], x[:, h + kv:])):
        done, row = [], 0
        for b, (p, t) in enumerate(zip(held, fresh)):
            for o in range(p // page, (p + t - 1) // page + 1):
                lo, hi = max(p, o * page), min(p + t, (o + 1) * page)
                i, a, z = int(s["table"][b, o]), lo - o * page, hi - o * page
                part = new[row + lo - p:row + hi - p].transpose(0, 1)
                need = torch.ceil(torch.log2(part.abs().amax((1, 2)) / 127)).clamp(min=-127)
                was = e[i].to(f64) - 127
                now = need if a == 0 else torch.maximum(need, was)
                c = codes[i].to(f64)
                c[:, :a] = torch.round(c[:, :a] * torch.exp2(was - now)[:, None, None])
                c[:, a:z] = torch.round(part * torch.exp2(-now)[:, None, None])
                done.append(c * torch.exp2(now)[:, None, None])
            row += t
        both.append(torch.stack(done))
    return {"q": x[:, :h], "k": both[0], "v": both[1]}
