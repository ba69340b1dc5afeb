"""The operators of a block's attention half, served from a quantised cache:
rotary positions and their gradient, the cache written and read back, and
attention over the cache.

Each case runs one pass through one of them, in its plain form (elementary
torch operations in 32 bits; angles, and keys on their way to 8 bits, in 64) or, where `own` is true, through the
framework's calls.  Shapes: 32 query heads over 8 key/value heads of 128 are
the Max-like stack's (batch 8 x 4096 tokens); the others are small or odd ones.

The cache: pages of `block` tokens; k codes [pages, kv heads, block, D], v codes
[pages, kv heads, D, block] (transposed), int8 or e4m3, one scale for each page
and kv head: the smallest power of two that holds the block's largest magnitude.  `kv_lens` counts a sequence's tokens, the new ones included;
row r of a batch belongs to sequence b where cu_q[b] <= r < cu_q[b + 1].
"""
import importlib
import math
import random

import numpy as np
import torch

own = False

QMAX = {"int8": 127.0, "e4m3": 448.0}
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _attention():
    return importlib.import_module("noor_-_bangla_ai_b200").attention


# ---------------------------------------------------------------- cases


def _case(name, op, **kw):
    c = {"name": name, "op": op, "dtype": "bf16", "Hq": 32, "Hkv": 8, "D": 128, "rot": 128, "layout": "interleaved",
         "stretch": 1.0, "block": 64, "fmt": "int8", "B": 1, "old": 0, "new": 1, "ragged": False, "window": 0,
         "T": 0, "pos": 0, "grad": False}
    c.update(kw)
    return c


def listed():
    return [
        # one decode step of 64 streams: q and k of one token each, far into their contexts
        _case("rope_decode", "rope", T=64, pos=30000),
        # a training batch of the Max-like stack (8 x 4096 tokens), forward and gradient
        _case("rope_train", "rope", T=32768, layout="half", grad=True),
        # part of an odd head rotated, in 32 bits, with frequencies stretched for a long context
        _case("rope_part_f32", "rope", dtype="f32", T=5003, Hq=12, Hkv=4, D=80, rot=20, stretch=8.0, pos=900000,
              grad=True),
        # a decode step of 128 streams into part-filled blocks
        _case("write_decode", "write", B=128, old=4000, new=1, ragged=True),
        # prompts of ragged lengths written at once
        _case("write_prompt", "write", B=8, old=0, new=4096, ragged=True, fmt="e4m3", block=32, layout="half"),
        # a 32-bit layer with odd heads, appended in the middle of blocks
        _case("write_f32_odd", "write", dtype="f32", B=5, old=333, new=77, ragged=True, Hq=9, Hkv=3, D=80, rot=40,
              block=16, layout="half"),
        # a cached prefix read back as the layer's own type
        _case("read_prefix", "read", B=32, old=4096, ragged=True),
        # one stream, one token, a short context: latency
        _case("attend_one", "attend", B=1, old=1000, new=1),
        # ragged decode batch of the Max-like stack
        _case("attend_batch", "attend", B=64, old=8192, new=1, ragged=True, fmt="e4m3"),
        # few streams over long contexts
        _case("attend_long", "attend", B=4, old=131072, new=1),
        # drafted tokens of several streams checked at once, sliding window, 32-bit layer
        _case("attend_draft_f32", "attend", dtype="f32", B=24, old=5000, new=7, ragged=True, window=1024, Hq=16,
              Hkv=4, D=64, rot=64, block=32),
        # prompt chunks on top of cached context
        _case("attend_prompt", "attend", B=2, old=6144, new=2048),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: operator, type, heads, format and block at random, sizes
    spread over their logarithm."""
    op = rng.choice(["rope", "write", "read", "attend", "attend"])
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (16, 16), (8, 1), (12, 4), (9, 3), (16, 2), (40, 8)])
    D = rng.choice([64, 80, 96, 128, 128, 256])
    c = _case("", op, dtype=rng.choice(["bf16", "bf16", "f32"]), Hq=Hq, Hkv=Hkv, D=D,
              rot=rng.choice([D, D, D // 4 // 2 * 2, D // 2]), layout=rng.choice(["interleaved", "half"]),
              stretch=rng.choice([1.0, 1.0, 4.0]), block=rng.choice([16, 32, 64]), fmt=rng.choice(["int8", "e4m3"]),
              ragged=rng.random() < 0.7)
    del c["name"]
    if op == "rope":
        c.update(T=_log(rng, 1, 16000), pos=_log(rng, 1, 1000000), grad=rng.random() < 0.5)
        return c
    budget = 4 * 10 ** 8 // (Hkv * D * 2)  # cached tokens in all
    B = _log(rng, 1, 96)
    if op == "write":
        c.update(B=B, old=_log(rng, 1, 8192), new=rng.choice([1, 1, _log(rng, 1, 2048)]))
        if B * c["new"] * Hkv * D > 2 ** 25:
            c["new"] = max(1, 2 ** 25 // (B * Hkv * D))
        c["old"] = max(1, min(c["old"], budget // B))
        return c
    c.update(B=B, old=max(1, min(_log(rng, 1, 100000), budget // B)))
    if op == "attend":
        c.update(new=rng.choice([1, 1, 1, _log(rng, 1, 16), _log(rng, 1, 1024)]),
                 window=rng.choice([0, 0, 0, _log(rng, 1, 2048)]))
        # scores of all rows: at most a sixteenth of the largest listed case's
        while c["new"] > 1 and B * Hq * c["new"] * (c["old"] + c["new"]) > 2 ** 26:
            c["new"] //= 2
    return c


def _lens(case):
    """(tokens cached before, new tokens) of each sequence.  Ragged batches of 8
    or more have an idle slot without new tokens."""
    B, old, new = case["B"], case["old"], case["new"]
    if not case["ragged"]:
        return [old] * B, [new] * B
    rng = random.Random(B * 1000003 + old * 1009 + new)
    olds = [rng.randint(old // 3, old) for _ in range(B)]
    news = [rng.randint(max(1, new // 3), new) for _ in range(B)]
    olds[0], news[0] = old, new
    if B >= 8:
        news[B // 2] = 0
    return olds, news


def _starts(case):
    """First token of each sequence that `read` reads."""
    olds, _ = _lens(case)
    return [n // 7 if case["ragged"] else 0 for n in olds]


def _inv_freq(case):
    i = np.arange(case["rot"] // 2, dtype=np.float64)
    return (10000.0 ** (-2.0 * i / max(case["rot"], 1)) / case["stretch"]).astype(np.float32)


# ---------------------------------------------------------------- inputs


def _scale_for(amax, fmt):
    """Smallest power of two s >= 2^-126 with amax <= Q s."""
    m, e = torch.frexp(amax.double())  # amax = m 2^e, m in [1/2, 1)
    q, qe = math.frexp(QMAX[fmt])
    e = e - qe + (m > q).to(e.dtype)
    return torch.where(amax > 0, torch.exp2(e.clamp(min=-126).double()), 2.0 ** -126).float()


def _quantised_pool(case, pages, gen):
    """Random cache contents: normal values with channels of different size,
    quantised page by page."""
    H, D, blk, fmt = case["Hkv"], case["D"], case["block"], case["fmt"]
    out = []
    for kind in ("k", "v"):
        shape = (pages, H, blk, D) if kind == "k" else (pages, H, D, blk)
        codes = torch.empty(shape, dtype=torch.int8 if fmt == "int8" else torch.float8_e4m3fn, device="cuda")
        scale = torch.empty((pages, H), device="cuda")
        gain = 0.5 + torch.rand((1, H, 1, D) if kind == "k" else (1, H, D, 1), device="cuda", generator=gen)
        step = max(1, 2 ** 27 // (H * blk * D))
        for p in range(0, pages, step):
            n = min(step, pages - p)
            x = torch.randn((n,) + shape[1:], device="cuda", generator=gen) * gain
            s = _scale_for(x.abs().amax((2, 3)), fmt)
            x = x / s[:, :, None, None]
            codes[p:p + n] = x.round().to(torch.int8) if fmt == "int8" else x.to(torch.float8_e4m3fn)
            scale[p:p + n] = s
        out += [codes, scale]
    return out


def _rows(counts):
    """For ragged rows: sequence of each row and its index there."""
    b = np.repeat(np.arange(len(counts)), counts)
    i = np.concatenate([np.arange(n) for n in counts]) if len(counts) else np.zeros(0)
    return torch.from_numpy(b.astype(np.int64)).cuda(), torch.from_numpy(i.astype(np.int64)).cuda()


def _cu(counts):
    return torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    Hq, Hkv, D, blk = case["Hq"], case["Hkv"], case["D"], case["block"]
    st = {"case": case}
    rand = lambda *shape: torch.randn(shape, device="cuda", generator=gen)
    inv = torch.from_numpy(_inv_freq(case)).cuda()
    st["inv_freq"] = inv
    if own:
        st["rotary"] = _attention().Rotary(inv, layout=case["layout"])
    if case["op"] == "rope":
        T = case["T"]
        st["positions"] = (torch.arange(T, device="cuda") + case["pos"]).to(torch.int32)
        st["q"], st["k"] = rand(T, Hq, D).to(dt), rand(T, Hkv, D).to(dt)
        if case["grad"]:
            st["gq"], st["gk"] = rand(T, Hq, D).to(dt), rand(T, Hkv, D).to(dt)
            if own:
                st["q"].requires_grad_(True)
                st["k"].requires_grad_(True)
        return st
    olds, news = _lens(case)
    if case["op"] == "read":
        news = [0] * len(olds)
    lens = [o + n for o, n in zip(olds, news)]
    used = [(n + blk - 1) // blk for n in lens]
    pages = sum(used) + 3
    order = torch.randperm(pages, device="cuda", generator=gen)
    table = torch.full((case["B"], max(max(used), 1)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    st["block_table"], st["kv_lens"] = table, torch.tensor(lens, dtype=torch.int32, device="cuda")
    st["k_codes"], st["k_scale"], st["v_codes"], st["v_scale"] = _quantised_pool(case, pages, gen)
    if own:
        st["cache"] = _attention().KVCache.from_tensors(st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"])
    if case["op"] == "read":
        starts = _starts(case)
        counts = [n - s for n, s in zip(lens, starts)]
        st["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        st["cu"], st["total"] = _cu(counts), sum(counts)
        st["row_b"], st["row_i"] = _rows(counts)
        return st
    N = sum(news)
    st["cu_q"], st["max_q"] = _cu(news), max(news)
    st["row_b"], st["row_i"] = _rows(news)
    if case["op"] == "attend":
        st["q"] = (2.5 * rand(N, Hq, D)).to(dt)
        return st
    # write: the new tokens, and the range of each sequence's touched blocks to read back
    st["q"], st["k"], st["v"] = rand(N, Hq, D).to(dt), (1.1 * rand(N, Hkv, D)).to(dt), rand(N, Hkv, D).to(dt)
    starts = [o // blk * blk for o in olds]
    counts = [n - s if new else 0 for n, s, new in zip(lens, starts, news)]
    st["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    st["cu"], st["total"] = _cu(counts), sum(counts)
    st["read_b"], st["read_i"] = _rows(counts)
    # the touched blocks, numbered: page, tokens it held before, block of each new token
    first, pos = [], []
    tasks = 0
    held = []
    task_b, task_j = [], []
    for b, (o, n) in enumerate(zip(olds, news)):
        first.append(tasks)
        for j in range(o // blk, (o + n - 1) // blk + 1 if n else o // blk):
            held.append(max(0, min(blk, o - j * blk)))
            task_b.append(b)
            task_j.append(j)
            tasks += 1
        pos += list(range(o, o + n))
    dev = lambda xs: torch.tensor(xs, dtype=torch.int64, device="cuda")
    st["positions"] = dev(pos)
    st["held"] = dev(held)
    st["task_page"] = table[dev(task_b), dev(task_j)].long()
    old_t = dev(olds)
    st["token_task"] = dev(first)[st["row_b"]] + st["positions"] // blk - old_t[st["row_b"]] // blk
    st["token_slot"] = st["positions"] % blk
    return st


# ---------------------------------------------------------------- plain forms


def _rotate(x, positions, inv_freq, layout, sign=1.0, dtype=torch.float32):
    """First 2 * len(inv_freq) dims of x [T, H, D] rotated, in `dtype`."""
    rot = 2 * inv_freq.numel()
    xf = x.to(dtype)
    if rot == 0:
        return xf
    ang = positions.double()[:, None] * inv_freq.double()[None, :]
    cos, sin = torch.cos(ang).to(dtype)[:, None], (sign * torch.sin(ang)).to(dtype)[:, None]
    y = xf.clone()
    if layout == "interleaved":
        a, b = xf[..., 0:rot:2], xf[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = xf[..., :rot // 2], xf[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * cos - b * sin, a * sin + b * cos
    return y


def _round8(x, fmt):
    """x f64 rounded to the values that a code stands for, ties to even."""
    if fmt == "int8":
        return x.round().clamp(-127, 127)
    _, e = torch.frexp(x)
    step = torch.exp2((e - 4).clamp(min=-9).double())
    return ((x / step).round() * step).clamp(-448, 448)


def _plain_rope(st):
    case, inv, pos = st["case"], st["inv_freq"], st["positions"]
    out = [_rotate(st[n], pos, inv, case["layout"]).to(st[n].dtype) for n in ("q", "k")]
    if case["grad"]:
        out += [_rotate(st[n], pos, inv, case["layout"], -1.0).to(st[n].dtype) for n in ("gq", "gk")]
    return out


def _append(codes, scale, x, st, transposed):
    """x [N, H, D] f64 into the touched blocks of one pool.  A block that held
    tokens keeps its scale or grows it, its codes rounded again."""
    case = st["case"]
    blk, fmt = case["block"], case["fmt"]
    pages, held = st["task_page"], st["held"]
    dense = torch.zeros((pages.numel(), case["Hkv"], blk, case["D"]), dtype=x.dtype, device=x.device)
    dense[st["token_task"], :, st["token_slot"]] = x
    s_old = torch.where(held[:, None] > 0, scale[pages], torch.zeros_like(scale[pages]))
    s = torch.maximum(s_old, _scale_for(dense.abs().amax((2, 3)), fmt))
    raw = codes.view(torch.int8)[pages]
    was = raw.view(codes.dtype).float()
    if transposed:
        raw, was = raw.transpose(2, 3), was.transpose(2, 3)
    slot = torch.arange(blk, device=x.device)[None, :]
    new = torch.where((slot < held[:, None])[:, None, :, None], was * s_old[:, :, None, None], dense)
    new = _round8(new / s[:, :, None, None], fmt).to(codes.dtype).view(torch.int8)
    valid = slot < held[:, None]
    valid[st["token_task"], st["token_slot"]] = True
    new = torch.where(valid[:, None, :, None], new, raw)
    codes.view(torch.int8)[pages] = new.transpose(2, 3) if transposed else new
    scale[pages] = s


def _gather(codes, scale, st, row_b, pos, transposed):
    """Values [rows, H, D] f32 of the tokens at `pos` of sequences row_b."""
    blk = st["case"]["block"]
    page = st["block_table"][row_b, pos // blk].long()
    slot = pos % blk
    raw = codes.view(torch.int8)
    raw = raw[page, :, :, slot] if transposed else raw[page, :, slot]
    return raw.view(codes.dtype).float() * scale[page][:, :, None]


def _plain_write(st):
    case = st["case"]
    q = _rotate(st["q"], st["positions"], st["inv_freq"], case["layout"]).to(st["q"].dtype)
    k = _rotate(st["k"], st["positions"], st["inv_freq"], case["layout"], dtype=torch.float64)
    _append(st["k_codes"], st["k_scale"], k, st, False)
    _append(st["v_codes"], st["v_scale"], st["v"].double(), st, True)
    pos = st["starts"].long()[st["read_b"]] + st["read_i"]
    return [q, _gather(st["k_codes"], st["k_scale"], st, st["read_b"], pos, False).to(q.dtype),
            _gather(st["v_codes"], st["v_scale"], st, st["read_b"], pos, True).to(q.dtype)]


def _plain_read(st):
    dt = DTYPES[st["case"]["dtype"]]
    pos = st["starts"].long()[st["row_b"]] + st["row_i"]
    return [_gather(st["k_codes"], st["k_scale"], st, st["row_b"], pos, False).to(dt),
            _gather(st["v_codes"], st["v_scale"], st, st["row_b"], pos, True).to(dt)]


def _plain_attend(st):
    case = st["case"]
    B, Hq, Hkv, D, n = case["B"], case["Hq"], case["Hkv"], case["D"], st["max_q"]
    g = Hq // Hkv
    table = st["block_table"].clamp(min=0).long()
    L = table.shape[1] * case["block"]
    k = st["k_codes"].view(torch.int8)[table].view(st["k_codes"].dtype).float()  # [B, pages, Hkv, block, D]
    k = (k * st["k_scale"][table][..., None, None]).transpose(1, 2).reshape(B, Hkv, L, D)
    v = st["v_codes"].view(torch.int8)[table].view(st["v_codes"].dtype).float()  # [B, pages, Hkv, D, block]
    v = (v * st["v_scale"][table][..., None, None]).permute(0, 2, 1, 4, 3).reshape(B, Hkv, L, D)
    q = torch.zeros((B, n, Hq, D), device=k.device)
    q[st["row_b"], st["row_i"]] = st["q"].float()
    q = q.view(B, n, Hkv, g, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, g * n, D)
    s = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    new = st["cu_q"][1:] - st["cu_q"][:-1]
    at = (st["kv_lens"] - new)[:, None] + torch.arange(n, device=k.device)[None, :]  # position of each row
    key = torch.arange(L, device=k.device)
    seen = key[None, None, :] <= at[:, :, None]
    if case["window"] > 0:
        seen &= at[:, :, None] - key[None, None, :] <= case["window"]
    seen = seen[:, None, None].expand(B, 1, g, n, L).reshape(B, 1, g * n, L)
    s = s.masked_fill(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top.isinf(), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.view(B, Hkv, g, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D)
    return o[st["row_b"], st["row_i"]].to(st["q"].dtype)


# ---------------------------------------------------------------- one pass


def run(state):
    st = state
    case = st["case"]
    if not own:
        return {"rope": _plain_rope, "write": _plain_write, "read": _plain_read, "attend": _plain_attend}[case["op"]](st)
    A = _attention()
    if case["op"] == "rope":
        q, k = A.rope_apply(st["q"], st["positions"], st["rotary"], k=st["k"])
        if case["grad"]:
            return [q.detach(), k.detach(), *torch.autograd.grad((q, k), (st["q"], st["k"]), (st["gq"], st["gk"]))]
        return [q, k]
    if case["op"] == "write":
        q = st["cache"].append(st["k"], st["v"], st["block_table"], st["kv_lens"], st["cu_q"], rotary=st["rotary"],
                               q=st["q"])
        return [q, *st["cache"].read(st["block_table"], st["starts"], st["cu"], st["total"],
                                      dtype=DTYPES[case["dtype"]])]
    if case["op"] == "read":
        return list(st["cache"].read(st["block_table"], st["starts"], st["cu"], st["total"],
                                     dtype=DTYPES[case["dtype"]]))
    return st["cache"].attention(st["q"], st["block_table"], st["kv_lens"], st["cu_q"], st["max_q"],
                                 window=case["window"])


# ---------------------------------------------------------------- work


def _visible(case):
    """(distinct cached tokens read, (row, key) pairs) over the batch."""
    olds, news = _lens(case)
    w = case["window"]
    tokens = pairs = 0
    for o, n in zip(olds, news):
        if n == 0:
            continue
        tokens += o + n - (max(0, o - w) if w else 0)
        for i in range(n):
            pairs += min(o + i + 1, w + 1) if w else o + i + 1
    return tokens, pairs


def work(case):
    b = 2 if case["dtype"] == "bf16" else 4
    Hq, Hkv, D, blk = case["Hq"], case["Hkv"], case["D"], case["block"]
    cached = 2.0 * Hkv * (D + 4.0 / blk)  # k and v of one token with their share of the scales
    if case["op"] == "rope":
        n = case["T"] * (Hq + Hkv) * (2 if case["grad"] else 1)
        return {"bytes": 2.0 * n * D * b + 4 * case["T"], "flops": 3.0 * n * case["rot"]}
    olds, news = _lens(case)
    if case["op"] == "read":
        n = sum(olds) - sum(_starts(case))
        return {"bytes": n * (cached + 2.0 * Hkv * D * b), "flops": 2.0 * n * Hkv * D}
    N = sum(news)
    if case["op"] == "write":
        back = sum(o + n - o // blk * blk for o, n in zip(olds, news) if n)
        return {"bytes": 2.0 * N * Hq * D * b + N * (2.0 * Hkv * D * b + cached) + back * (cached + 2.0 * Hkv * D * b),
                "flops": N * (3.0 * (Hq + Hkv) * case["rot"] + 4.0 * Hkv * D) + back * 2.0 * Hkv * D}
    tokens, pairs = _visible(case)
    return {"bytes": tokens * cached + 2.0 * N * Hq * D * b, "flops": 4.0 * D * Hq * pairs}


# ---------------------------------------------------------------- in 64 bits


def _turn64(x, pos, inv, layout, sign):
    """Rotation as a complex product, in 64 bits."""
    half = inv.numel()
    x = x.double()
    if half == 0:
        return x
    head, rest = x[..., :2 * half], x[..., 2 * half:]
    pair = head.unflatten(-1, (half, 2)) if layout == "interleaved" else head.unflatten(-1, (2, half)).transpose(-1, -2)
    ang = sign * pos.double().unsqueeze(-1) * inv.double()
    z = torch.view_as_complex(pair.contiguous()) * torch.polar(torch.ones_like(ang), ang).unsqueeze(1)
    pair = torch.view_as_real(z)
    head = (pair if layout == "interleaved" else pair.transpose(-1, -2)).flatten(-2)
    return torch.cat([head, rest], -1)


def _grid64(x, fmt):
    """The nearest of a format's values to each x, found in their list; a tie
    goes to the even code."""
    if fmt == "int8":
        vals = torch.arange(128, dtype=torch.float64, device=x.device)
    else:
        vals = torch.arange(127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
    mid = (vals[1:] + vals[:-1]) / 2
    i = torch.searchsorted(mid, x.abs().contiguous())
    tie = (x.abs() == mid[i.clamp(max=mid.numel() - 1)]) & (i < mid.numel()) & (i % 2 == 1)
    return vals[i + tie] * x.sign()


def _exact_pool(st, codes, scale, new, transposed):
    """Values after the append of the tokens to be read back, block by block."""
    case = st["case"]
    blk, qmax, fmt = case["block"], QMAX[case["fmt"]], case["fmt"]
    old = codes.view(torch.int8)[st["task_page"]].view(codes.dtype).double()
    old = old.transpose(2, 3) if transposed else old
    s_old = scale[st["task_page"]].double() * (st["held"] > 0)[:, None]
    fresh = torch.zeros_like(old)
    fresh[st["token_task"], :, st["token_slot"]] = new
    need = torch.ceil(torch.log2(fresh.abs().flatten(2).max(-1).values / qmax)).clamp(min=-126)
    s = torch.maximum(s_old, torch.exp2(need))[:, :, None, None]
    kept = _grid64(old * (s_old[:, :, None, None] / s), fmt)
    wrote = _grid64(fresh / s, fmt)
    in_old = (torch.arange(blk, device=old.device) < st["held"][:, None])[:, None, :, None]
    vals = torch.where(in_old, kept, wrote) * s  # powers of two: exact
    # rows to read back are the touched blocks' tokens, in order
    count = st["held"].clone()
    count.index_add_(0, st["token_task"], torch.ones_like(st["token_task"]))
    keep = torch.arange(blk, device=old.device) < count[:, None]
    return vals.transpose(1, 2)[keep]


def exact(case, seed):
    st = prepare(case, seed)
    inv, layout = st["inv_freq"], case["layout"]
    if case["op"] == "rope":
        names = [("q", 1.0), ("k", 1.0)] + ([("gq", -1.0), ("gk", -1.0)] if case["grad"] else [])
        return [_turn64(st[n].detach(), st["positions"], inv, layout, s) for n, s in names]
    if case["op"] == "write":
        return [_turn64(st["q"], st["positions"], inv, layout, 1.0),
                _exact_pool(st, st["k_codes"], st["k_scale"], _turn64(st["k"], st["positions"], inv, layout, 1.0), False),
                _exact_pool(st, st["v_codes"], st["v_scale"], st["v"].double(), True)]
    blk, D = case["block"], case["D"]
    cu = st["cu" if case["op"] == "read" else "cu_q"].tolist()
    lens = st["kv_lens"].tolist()
    kc, vc = st["k_codes"].view(torch.int8), st["v_codes"].view(torch.int8)

    def cached(b, head, n):
        """k and v [n, D] of one sequence and kv head, in 64 bits."""
        pages = st["block_table"][b, :(n + blk - 1) // blk].long()
        k = kc[pages, head].view(st["k_codes"].dtype).double() * st["k_scale"][pages, head].double()[:, None, None]
        v = vc[pages, head].view(st["v_codes"].dtype).double() * st["v_scale"][pages, head].double()[:, None, None]
        return k.reshape(-1, D)[:n], v.transpose(1, 2).reshape(-1, D)[:n]

    if case["op"] == "read":
        k, v = (torch.empty((st["total"], case["Hkv"], D), dtype=torch.float64, device="cuda") for _ in range(2))
        for b, start in enumerate(_starts(case)):
            for h in range(case["Hkv"]):
                kk, vv = cached(b, h, lens[b])
                k[cu[b]:cu[b + 1], h], v[cu[b]:cu[b + 1], h] = kk[start:], vv[start:]
        return [k, v]
    out = torch.zeros((cu[-1], case["Hq"], D), dtype=torch.float64, device="cuda")
    g = case["Hq"] // case["Hkv"]
    for b in range(case["B"]):
        n = cu[b + 1] - cu[b]
        if n == 0:
            continue
        at = torch.arange(lens[b] - n, lens[b], device="cuda")[:, None]
        key = torch.arange(lens[b], device="cuda")[None, :]
        hidden = (key > at) | ((at - key > case["window"]) if case["window"] else torch.zeros_like(key > at))
        for h in range(case["Hkv"]):
            kk, vv = cached(b, h, lens[b])
            for i in range(g):
                s = (st["q"][cu[b]:cu[b + 1], h * g + i].double() @ kk.T) / math.sqrt(D)
                out[cu[b]:cu[b + 1], h * g + i] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ vv
    return out
