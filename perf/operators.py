"""The paged key / value cache and the attention over it: calls, plain forms, results in 64 bits and floors.

Two kinds of case.  "append": the new tokens' keys and values go into the pages of their sequences, the keys rotated on the way.  "attend": the
new tokens' queries see the positions of their sequence up to their own.  Either over pages of f16 numbers or of e4m3 numbers under one
power-of-two scale for each 16 positions and head.  A call takes a ragged batch: sequence s has rows row_start[s] .. row_start[s + 1] - 1 of it, at
positions pos0[s], pos0[s] + 1, ...; keys, values and queries are views of one projection's output.

listed() names twelve calls; draw() takes more from the same ranges.
"""
import math
import random

import torch

own = False
F64 = torch.float64
ACT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 16  # positions under one scale
E_MIN, E_MAX, E4M3_MAX = -15, 7, 448.0
# query heads, key / value heads and rotation of the benchmark configurations
HEADS = {"3b": (16, 2, 1, 1e6), "32b": (40, 8, 1, 1e6), "70b": (64, 8, 0, 5e5), "moe": (32, 4, 1, 1e6)}


def case(name, op, cache, act, shape, seqs, rows, past, page, dim=128, window=0, mix=1):
    """rows, past: (least, most) new and earlier tokens of a sequence; mix: the seed of the lengths"""
    n_head, n_kv, neox, theta = HEADS[shape]
    c = dict(op=op, cache=cache, act=act, n_head=n_head, n_kv=n_kv, neox=neox, theta=theta, dim=dim, seqs=seqs, rows_lo=rows[0], rows_hi=rows[1],
             past_lo=past[0], past_hi=past[1], page=page, window=window, mix=mix)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the smallest call: the new token of one user
        case("append_one_f16", "append", "f16", "f32", "32b", 1, (1, 1), (2047, 2047), 16),
        # a decode step of 64 users
        case("append_users_e4m3", "append", "e4m3", "f32", "70b", 64, (1, 1), (100, 8000), 16, mix=2),
        # a micro-batch of the usual size in the middle of a prompt
        case("append_prompt_f16", "append", "f16", "f32", "32b", 1, (512, 512), (1536, 1536), 64),
        # several long prompts of odd lengths that start inside a page
        case("append_prompts_e4m3", "append", "e4m3", "bf16", "70b", 6, (900, 5000), (1, 300), 32, mix=3),
        # the headline configuration's decode step: one user at context 2048
        case("attend_one_f16", "attend", "f16", "f32", "32b", 1, (1, 1), (2047, 2047), 16),
        # one user far into a long context
        case("attend_one_long_e4m3", "attend", "e4m3", "bf16", "70b", 1, (1, 1), (131000, 131000), 64),
        # 64 users of a mixture of experts with contexts of every length
        case("attend_users_f16", "attend", "f16", "f16", "moe", 64, (1, 1), (300, 9000), 16, mix=4),
        # the largest batch of users: 200 of them, in 8 bits, with 32-bit activations
        case("attend_users_e4m3", "attend", "e4m3", "f32", "32b", 200, (1, 1), (60, 6000), 32, mix=5),
        # drafts of up to four tokens checked at once, heads of 64, a sliding window
        case("attend_drafts_f16", "attend", "f16", "f32", "3b", 9, (1, 4), (500, 5000), 48, dim=64, window=1024, mix=6),
        # a micro-batch of the usual size in the middle of a prompt
        case("attend_prompt_f16", "attend", "f16", "f32", "32b", 1, (512, 512), (1536, 1536), 64),
        # decode steps and chunks of prompts in one call
        case("attend_mixed_e4m3", "attend", "e4m3", "bf16", "moe", 14, (1, 700), (0, 7000), 16, mix=7),
        # the largest: a chunk of a long prompt
        case("attend_long_prompt_f16", "attend", "f16", "bf16", "32b", 1, (4096, 4096), (12288, 12288), 128),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op, cache = rng.choice(("append", "attend")), rng.choice(("f16", "e4m3"))
    act, shape = rng.choice(("f32", "f32", "bf16", "f16")), rng.choice(sorted(HEADS))
    dim, page = rng.choice((128, 128, 128, 64)), rng.choice((16, 16, 32, 48, 64, 128, 256))
    window = log(64, 8192) if op == "attend" and rng.random() < 0.2 else 0
    mix = rng.randrange(1 << 20)
    if op == "append":
        if rng.random() < 0.5:
            seqs, rows = log(1, 256), (1, rng.choice((1, 1, 4)))
        else:
            seqs = log(1, 8)
            top = log(16, 20000 // seqs)
            rows = (max(1, top // rng.choice((1, 3, 10))), top)
        past = log(1, 8000)
        return case(None, op, cache, act, shape, seqs, rows, (past // rng.choice((1, 4, 50)), past), page, dim, mix=mix)
    kind = rng.random()
    if kind < 0.5:  # decode, up to 600 k positions over all sequences
        seqs = log(1, 200)
        past, rows = log(8, min(131000, 600000 // seqs)), (1, rng.choice((1, 1, 1, 4)))
    elif kind < 0.8:  # one or a few prompts
        seqs = log(1, 4)
        top = log(5, 4096 // seqs)
        rows, past = (max(1, top // rng.choice((1, 2, 5))), top), log(1, 8192 // seqs)
    else:  # both in one call
        seqs = log(3, 16)
        rows, past = (1, log(20, 500)), log(50, 6000)
    return case(None, op, cache, act, shape, seqs, rows, (past // rng.choice((1, 4, 30)), past), page, dim, window, mix)


def lengths(c):
    """new and earlier tokens of each sequence: the case's own, whatever the inputs"""
    r = random.Random(c["mix"])

    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(r.uniform(math.log(lo + 1), math.log(hi + 1))) - 1))))

    return [log(c["rows_lo"], c["rows_hi"]) for _ in range(c["seqs"])], [log(c["past_lo"], c["past_hi"]) for _ in range(c["seqs"])]


def work(c):
    rows, past = lengths(c)
    act, code = 4 if c["act"] == "f32" else 2, 2 if c["cache"] == "f16" else 1
    per_token, n = c["n_kv"] * c["dim"], sum(rows)
    if c["op"] == "append":
        blocks = sum((p + t - 1) // BLOCK - p // BLOCK + 1 for p, t in zip(past, rows))
        return {"bytes": 2 * n * per_token * (act + code) + (0 if code == 2 else blocks * c["n_kv"] * 16), "flops": 6 * n * per_token}
    pairs = keys = 0
    for p, t in zip(past, rows):
        w = c["window"] or p + t
        pairs += sum(min(p + i + 1, w) for i in range(t))
        keys += min(p + t, w + t - 1)
    return {"bytes": 2 * keys * per_token * code + (0 if code == 2 else 2 * keys // BLOCK * c["n_kv"] * 4) + 2 * n * c["n_head"] * c["dim"] * act,
            "flops": 4 * pairs * c["n_head"] * c["dim"]}


def scale_of(amax):
    """the smallest power of two that brings amax to at most the largest e4m3 number, within the exponents at which every code is an f16 number"""
    m, e = torch.frexp(amax)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(E_MIN, E_MAX)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, torch.full_like(e, E_MIN)))


def pool(c, n_pages, gen):
    """pages [n_pages][n_kv][page][dim] of what a model's layers put there, and scales [n_pages][n_kv][page / 16]"""
    shape = (n_pages, c["n_kv"], c["page"], c["dim"])
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16)
    if c["cache"] == "f16":
        return x, None
    x = x.reshape(n_pages, c["n_kv"], c["page"] // BLOCK, BLOCK * c["dim"])
    x *= 0.25 + torch.rand(x.shape[:3] + (1,), generator=gen, device="cuda", dtype=torch.float16)  # blocks are not all alike
    s = scale_of(x.abs().amax(-1).float())
    return (x / s[..., None].half()).to(torch.float8_e4m3fn).reshape(shape), s


def prepare(c, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    rows, past = lengths(c)
    pages = [(p + t + c["page"] - 1) // c["page"] for p, t in zip(past, rows)]
    n_pages = sum(pages) + 3
    perm = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32).cpu()
    table = torch.full((c["seqs"], max(pages)), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(pages):
        table[s, :n] = perm[at:at + n]
        at += n
    k_pages, k_scale = pool(c, n_pages, gen)
    v_pages, v_scale = pool(c, n_pages, gen)
    n, nh, nkv = sum(rows), c["n_head"], c["n_kv"]
    qkv = torch.randn((n, nh + 2 * nkv, c["dim"]), generator=gen, device="cuda")
    qkv[:, nh:nh + nkv, ::11] *= 3.0  # some channels of the keys stand out
    qkv = qkv.to(ACT[c["act"]])
    start = torch.tensor([0] + rows).cumsum(0).to(torch.int32)
    return dict(case=c, k_pages=k_pages, v_pages=v_pages, k_scale=k_scale, v_scale=v_scale, table=table.cuda(), row_start=start.cuda(),
                pos0=torch.tensor(past, dtype=torch.int32).cuda(), q=qkv[:, :nh], k=qkv[:, nh:nh + nkv], v=qkv[:, nh + nkv:],
                most=max(rows), longest=max(p + t for p, t in zip(past, rows)))


def run(s):
    c = s["case"]
    if own:
        from mesh_llm_b200 import ops

        if c["op"] == "append":
            ops.kv_pages_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["row_start"], s["pos0"], c["theta"], c["neox"],
                                k_scale=s["k_scale"], v_scale=s["v_scale"])
            return pages_of(s)
        return ops.attention_pages(s["q"], s["k_pages"], s["v_pages"], s["table"], s["row_start"], s["pos0"], s["most"], c["theta"], c["neox"],
                                   window=c["window"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    return append(s) if c["op"] == "append" else attend(s)


def pages_of(s):
    """the updated cache: f16 numbers, or e4m3 numbers and what each block of them is multiplied by"""
    return {n: s[n] for n in ("k_pages", "v_pages", "k_scale", "v_scale") if s[n] is not None}


def places(s):
    """sequence, position, page and place inside it of each row"""
    page, start = s["case"]["page"], s["row_start"].long()
    row = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.bucketize(row, start[1:], right=True)
    pos = s["pos0"].long()[seq] + row - start[seq]
    return seq, pos, s["table"].long()[seq, pos // page], pos % page


def rotate(x, pos, c):
    half = c["dim"] // 2
    angle = pos.to(F64)[:, None] * c["theta"] ** (-torch.arange(half, device="cuda", dtype=F64) / half)
    cos, sin = (f(angle).to(x.dtype)[:, None] for f in (torch.cos, torch.sin))
    a, b = (x[..., :half], x[..., half:]) if c["neox"] else (x[..., 0::2], x[..., 1::2])
    a, b = a * cos - b * sin, a * sin + b * cos
    return torch.cat((a, b), -1) if c["neox"] else torch.stack((a, b), -1).flatten(-2)


def append(s):
    c = s["case"]
    _, pos, page, place = places(s)
    for x, pages, scale in ((rotate(s["k"].float(), pos, c), s["k_pages"], s["k_scale"]), (s["v"].float(), s["v_pages"], s["v_scale"])):
        if scale is None:
            pages[page, :, place] = x.half()
            continue
        n_pages, n_kv, size, dim = pages.shape
        blocks = size // BLOCK
        block = page * blocks + place // BLOCK  # a row's block, among those of all pages
        amax = torch.zeros((n_pages * blocks, n_kv), device="cuda").index_reduce_(0, block, x.abs().amax(-1), "amax")
        first = torch.full((n_pages * blocks,), BLOCK, device="cuda").index_reduce_(0, block, place % BLOCK, "amin")
        old = scale.transpose(1, 2).reshape(-1, n_kv)
        new = torch.where((first > 0)[:, None], torch.maximum(old, scale_of(amax)), scale_of(amax))
        new = torch.where((first < BLOCK)[:, None], new, old)  # blocks without a new row stay
        codes = pages.view(n_pages, n_kv, blocks, BLOCK, dim)
        at = torch.unique(block)  # the rows that such blocks hold already, under the new scale
        ratio = (old / new)[at][:, :, None, None]
        held = torch.arange(BLOCK, device="cuda")[None, :] < first[at][:, None]
        was = codes.view(torch.uint8)[at // blocks, :, at % blocks].view(pages.dtype).float()
        codes.view(torch.uint8)[at // blocks, :, at % blocks] = torch.where(held[:, None, :, None], was * ratio, was).to(pages.dtype).view(torch.uint8)
        scale.copy_(new.view(n_pages, blocks, n_kv).transpose(1, 2))
        pages.view(torch.uint8)[page, :, place] = (x / new[block][..., None]).to(pages.dtype).view(torch.uint8)
    return pages_of(s)


def dense(pages, scale, table, dtype):
    """what the pages of each sequence hold: [sequences][n_kv][positions][dim]"""
    at = table.long().clamp(min=0)
    x = pages.view(torch.uint8)[at].view(pages.dtype).to(dtype) if scale is not None else pages[at].to(dtype)
    if scale is not None:
        x = x * scale[at].to(dtype).repeat_interleave(BLOCK, -1)[..., None]
    return x.transpose(1, 2).flatten(2, 3)


def attend(s):
    c = s["case"]
    dim, nkv, group = c["dim"], c["n_kv"], c["n_head"] // c["n_kv"]
    seq, pos, _, _ = places(s)
    t = torch.arange(s["q"].shape[0], device="cuda") - s["row_start"].long()[seq]  # a row's number within its sequence
    q = torch.zeros((c["seqs"], s["most"], nkv, group, dim), device="cuda")
    q[seq, t] = rotate(s["q"].float(), pos, c).unflatten(1, (nkv, group))
    q = q.permute(0, 2, 3, 1, 4).flatten(2, 3) / math.sqrt(dim)
    k, v = (dense(p, x, s["table"], torch.float32) for p, x in ((s["k_pages"], s["k_scale"]), (s["v_pages"], s["v_scale"])))
    p = (q @ k.transpose(-1, -2)).unflatten(2, (group, s["most"]))
    at = s["pos0"].long()[:, None, None] + torch.arange(s["most"], device="cuda")[:, None]
    key = torch.arange(k.shape[2], device="cuda")
    seen = key <= at
    if c["window"]:
        seen &= key > at - c["window"]
    p.masked_fill_(~seen[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v).unflatten(2, (group, s["most"])) / total
    return o.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, t].to(ACT[c["act"]])


def exact(c, seed):
    """The same from the definition in 64 bits, one sequence and head at a time."""
    s = prepare(c, seed)
    rows, past = lengths(c)
    half, page, group = c["dim"] // 2, c["page"], c["n_head"] // c["n_kv"]
    turn = torch.tensor([c["theta"] ** (-i / half) for i in range(half)], dtype=F64, device="cuda")

    def turned(x, pos):
        z = torch.polar(torch.ones((), dtype=F64, device="cuda"), pos.to(F64)[:, None, None] * turn)
        y = torch.complex(x[..., :half], x[..., half:]) if c["neox"] else torch.complex(x[..., 0::2].contiguous(), x[..., 1::2].contiguous())
        y = y * z
        return torch.cat((y.real, y.imag), -1) if c["neox"] else torch.view_as_real(y).flatten(-2)

    if c["op"] == "append":
        return exact_append(c, s, rows, past, turned)
    out = torch.empty(s["q"].shape, dtype=F64, device="cuda")
    at = 0
    for i, (t, p) in enumerate(zip(rows, past)):
        pos = torch.arange(p, p + t, device="cuda")
        low = max(0, p - c["window"] + 1) if c["window"] else 0
        key = torch.arange(low, p + t, device="cuda")
        where = s["table"][i].long()[key // page], key % page
        q = turned(s["q"][at:at + t].to(F64), pos)
        hidden = key > pos[:, None]
        if c["window"]:
            hidden |= key <= pos[:, None] - c["window"]
        for h in range(c["n_kv"]):
            k, v = (x[:, h].to(F64)[where] * (1 if f is None else f[where[0], h, where[1] // BLOCK].to(F64)[:, None])
                    for x, f in ((s["k_pages"], s["k_scale"]), (s["v_pages"], s["v_scale"])))
            for g in range(h * group, (h + 1) * group):
                w = torch.softmax((q[:, g] @ k.T / math.sqrt(c["dim"])).masked_fill_(hidden, -math.inf), -1)
                out[at:at + t, g] = w @ v
        at += t
    return out


def exact_append(c, s, rows, past, turned):
    page, found, at = c["page"], {}, 0
    for n in ("k", "v"):
        found[n + "_pages"] = s[n + "_pages"].to(F64)
        if s[n + "_scale"] is not None:
            found[n + "_scale"] = s[n + "_scale"].to(F64)
    for i, (t, p) in enumerate(zip(rows, past)):
        pos = torch.arange(p, p + t, device="cuda")
        new = {"k": turned(s["k"][at:at + t].to(F64), pos), "v": s["v"][at:at + t].to(F64)}
        at += t
        where = s["table"][i].long()[pos // page]
        for n, x in new.items():
            pages, scale = found[n + "_pages"], found.get(n + "_scale")
            if scale is None:
                pages[where, :, pos % page] = x
                continue
            b0, b1 = p // BLOCK, (p + t - 1) // BLOCK + 1  # the sequence's blocks with new rows
            grid = torch.zeros(((b1 - b0) * BLOCK,) + x.shape[1:], dtype=F64, device="cuda")
            grid[p - b0 * BLOCK:p - b0 * BLOCK + t] = x
            grid = grid.unflatten(0, (b1 - b0, BLOCK))
            top = grid.abs().amax((1, 3))
            f = 2.0 ** torch.ceil(torch.log2(top / E4M3_MAX)).clamp(E_MIN, E_MAX)
            b = torch.arange(b0, b1, device="cuda")
            pg, in_page = s["table"][i].long()[b * BLOCK // page], b * BLOCK % page // BLOCK
            if p % BLOCK:
                f[0] = torch.maximum(f[0], scale[pg[0], :, in_page[0]])
                held = slice(int(in_page[0]) * BLOCK, int(in_page[0]) * BLOCK + p % BLOCK)
                pages[pg[0], :, held] *= (scale[pg[0], :, in_page[0]] / f[0])[:, None, None]
            scale[pg, :, in_page] = f
            pages[where, :, pos % page] = x / f[pos // BLOCK - b0][..., None]
    return found
