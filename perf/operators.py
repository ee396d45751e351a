"""Measured work of the operators on a paged KV pool held in 4 bits: writing tokens into it, reading them back, decode and
prefill attention over it.

The pool is four U8 tensors: codes [pages, KV heads, page, head / 2] of K and of V, two 4-bit floats (e2m1: sign, two bits of
exponent, one of mantissa; magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6) per byte, the even element in the low half, and scales
[pages, KV heads, page, head / 32], one exponent (bias 127) for each 32 elements. A group is written with the exponent of its
largest magnitude less two, kept within 2^-23 .. 2^13, elements rounded to the nearest (ties to the even code) and held at 6;
a group with a value that is not finite is written as scale 255, and reads as NaN.

Families (``case["op"]``):

* ``write_read`` - new K / V tokens written into their slots, then read back from there (``paged_caching_fp4``,
                   ``paged_reading_fp4``): what a chunk does whose attention shall see the same values as later steps
* ``read``       - tokens read out of the pool (``paged_reading_fp4``)
* ``decode``     - one query token per sequence over the pool (``paged_attention_fp4``)
* ``prefill``    - runs of new tokens over their history and themselves (``paged_attention_prefill_fp4``)

Where ``own`` is false the same is computed with elementary torch operations in 32 bits. The lengths of a batch are fixed by
the case (a stratified draw between its bounds), the seed decides which sequence has which, where its pages lie, and every value.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_INDEX = {"i64": torch.int64, "i32": torch.int32}
_GROUP = 32                    # elements under one scale
_LEAST, _MOST = 127 - 23, 127 + 13  # scales that are written
_SPARE_PAGES = 0.10            # of the pool, as a server keeps them free
_MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _case(name, op, **more):
    c = dict(name=name, op=op, dtype="bf16", index="i64", page=16, alibi=False, heads=32, kv_heads=8, head=128)
    c.update(more)
    return c


def listed():
    return [
        # a single user's chat: the new token of one layer; latency is all there is
        _case("write_read_one", "write_read", tokens=1, padding=0.0),
        # a serving chunk, some of its tokens padding
        _case("write_read_4096", "write_read", tokens=4096, padding=0.05),
        # an older multi-head model's prompt: heads of 64, fp16, pages of 32, an odd count
        _case("write_read_mha64_1531", "write_read", dtype="fp16", page=32, tokens=1531, padding=0.0, heads=16, kv_heads=16,
              head=64),
        # one conversation's history handed to another program
        _case("read_history_1023", "read", dtype="fp16", tokens=1023, padding=0.0),
        # a long shared document read back for a chunk of another precision
        _case("read_document_65536", "read", tokens=65536, padding=0.0),
        # the same single user's attention; launches and latency
        _case("decode_one", "decode", seqs=1, min_len=1023, max_len=1023),
        # the ordinary serving batch: 8B-class GQA decode, ragged lengths
        _case("decode_gqa_b32", "decode", seqs=32, min_len=512, max_len=4096),
        # multi-head, no grouping, heads of 64, ALiBi, 32-bit tables, pages of 32, short odd lengths
        _case("decode_mha64_alibi_b19", "decode", dtype="fp16", index="i32", page=32, alibi=True, seqs=19, heads=16,
              kv_heads=16, head=64, min_len=37, max_len=1531),
        # the largest decode call: a 70B-class share of a big batch, fp16
        _case("decode_share_b128", "decode", dtype="fp16", seqs=128, heads=64, min_len=1024, max_len=8192),
        # a few drafted tokens of each sequence checked at once over their histories
        _case("prefill_drafts_b8", "prefill", seqs=8, min_new=3, max_new=5, min_hist=2000, max_hist=6000),
        # whole prompts
        _case("prefill_prompts_b4", "prefill", seqs=4, min_new=1000, max_new=2500, min_hist=0, max_hist=0),
        # chunks over a long history (chunked prefill)
        _case("prefill_chunked_b16", "prefill", seqs=16, min_new=128, max_new=512, min_hist=1024, max_hist=8192),
    ]


# ---- drawn cases: the same families over their whole ranges ----

_LAYOUTS = [(32, 8), (32, 8), (64, 8), (8, 8), (40, 8), (16, 16), (48, 8), (28, 4), (8, 1)]  # query / KV heads


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _span(rng, lo, hi):
    """A lower and an upper bound inside [lo, hi], at most a factor of eight apart."""
    top = _log_int(rng, lo, hi)
    return max(lo, int(top * rng.uniform(0.125, 1.0))), top


def _drawn(rng):
    c = dict(op=rng.choice(["write_read", "read", "decode", "decode", "decode", "prefill", "prefill"]),
             index=rng.choice(["i64", "i64", "i32"]), page=rng.choice([16, 16, 16, 32, 64, 128, 8, 24]),
             head=rng.choice([64, 128, 128, 128, 192, 256]), alibi=False)
    c["heads"], c["kv_heads"] = rng.choice(_LAYOUTS)
    if c["op"] in ("write_read", "read"):
        c["dtype"] = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        c["tokens"] = _log_int(rng, 1, 16384 if c["op"] == "write_read" else 65536)
        c["padding"] = rng.choice([0.0, 0.05])
        return c
    c["dtype"] = rng.choice(["bf16", "bf16", "fp16"])
    c["alibi"] = rng.random() < 0.15
    if c["op"] == "decode":
        c["seqs"] = _log_int(rng, 1, 256)
        c["min_len"], c["max_len"] = _span(rng, 1, 32768)
    else:
        c["seqs"] = _log_int(rng, 1, 32)
        c["min_new"], c["max_new"] = _span(rng, 1, 4096)
        c["min_hist"], c["max_hist"] = (0, 0) if rng.random() < 0.4 else _span(rng, 16, 8192)
    return c


def draw(rng: random.Random):
    while True:
        c = _drawn(rng)
        w = work(c)
        # no more than the largest listed cases: the decode share's bytes, the chunks' products and padded scores
        if w["bytes"] <= 6.4e8 and w["flops"] <= 2.5e11:
            if c["op"] != "prefill" or c["seqs"] * c["heads"] * c["max_new"] * (c["max_new"] + c["max_hist"]) <= 2.3e9:
                return c


# ---- lengths and work: functions of the case alone ----

def _stratified(count, lo, hi, salt):
    """``count`` lengths spread over [lo, hi]: one from each of as many equal parts, in no particular order."""
    rng = random.Random("%d %d %d %d" % (count, lo, hi, salt))
    got = [lo + int((i + rng.random()) / count * (hi - lo + 1)) for i in range(count)]
    rng.shuffle(got)
    return got


def _lengths(case):
    """(new tokens, tokens seen at the end of the pass) of every sequence."""
    if case["op"] == "decode":
        return [1] * case["seqs"], _stratified(case["seqs"], case["min_len"], case["max_len"], 1)
    new = _stratified(case["seqs"], case["min_new"], case["max_new"], 2)
    hist = _stratified(case["seqs"], case["min_hist"], case["max_hist"], 3)
    return new, [n + h for n, h in zip(new, hist)]


def _padding_tokens(case):
    return int(case["tokens"] * case["padding"])


def _held_bytes(case):
    """Of one token's K and V in the pool."""
    return 2 * case["kv_heads"] * (case["head"] // 2 + case["head"] // _GROUP)


def work(case):
    head, heads, kv = case["head"], case["heads"], case["kv_heads"]
    if case["op"] in ("write_read", "read"):
        wide = 2 * kv * head * (4 if case["dtype"] == "fp32" else 2)
        tokens, valid = case["tokens"], case["tokens"] - _padding_tokens(case)
        b = valid * _held_bytes(case) + tokens * (wide + 8)  # read back
        if case["op"] == "write_read":
            b += valid * (wide + _held_bytes(case))
        return {"bytes": b, "flops": 0}
    new, total = _lengths(case)
    item = 8 if case["index"] == "i64" else 4
    pages = sum(-(-t // case["page"]) for t in total)
    b = sum(total) * _held_bytes(case) + sum(new) * heads * head * 4 + (pages + 2 * len(new)) * item
    pairs = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, total))
    return {"bytes": b, "flops": pairs * heads * 4 * head}


# ---- the plain form ----

def _quantised(x):
    """(codes [.., n / 2], scales [.., n / 32]) of x [.., n]."""
    groups = x.float().unflatten(-1, (-1, _GROUP))
    exponent = groups.abs().amax(-1).view(torch.int32) >> 23
    scales = torch.where(exponent == 255, 255, (exponent - 2).clamp(_LEAST, _MOST))
    unit = ((254 - scales) << 23).view(torch.float32)  # 1 / 2^(scale - 127); a power of two, so the product is exact
    a = groups.abs() * unit[..., None]
    codes = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int()
             + (a >= 3.5).int() + (a > 5.0).int())
    codes = codes + 8 * torch.signbit(groups).int()
    codes = torch.where((scales == 255)[..., None], 0, codes).flatten(-2)
    return (codes[..., 0::2] + 16 * codes[..., 1::2]).to(torch.uint8), scales.to(torch.uint8)


def _values(codes, scales):
    """The values that codes [.., n / 2] under scales [.., n / 32] stand for, in 32 bits."""
    table = torch.tensor(_MAGNITUDES + tuple(-m for m in _MAGNITUDES), device=codes.device)
    pairs = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)
    unit = (scales.int() << 23).view(torch.float32)
    unit = torch.where(scales == 255, math.nan, unit)
    return (table[pairs.int()].unflatten(-1, (-1, _GROUP)) * unit[..., None]).flatten(-2)


def _rows(pool, page, row):
    return pool[page, :, row]


def _read(s):
    slots, block = s["slots"], s["case"]["page"]
    page, row = slots.clamp(min=0) // block, slots.clamp(min=0) % block
    held = (slots >= 0)[:, None, None]
    k = _values(_rows(s["k_codes"], page, row), _rows(s["k_scales"], page, row))
    v = _values(_rows(s["v_codes"], page, row), _rows(s["v_scales"], page, row))
    return torch.where(held, k, 0.0).to(s["dtype"]), torch.where(held, v, 0.0).to(s["dtype"])


def _write(s):
    held = s["slots"] >= 0
    slots, block = s["slots"][held], s["case"]["page"]
    page, row = slots // block, slots % block
    s["k_codes"][page, :, row], s["k_scales"][page, :, row] = _quantised(s["k"][held])
    s["v_codes"][page, :, row], s["v_scales"][page, :, row] = _quantised(s["v"][held])


def _attention(s):
    """Every sequence's queries, padded to the longest run, over its tokens, padded to the table's width."""
    case = s["case"]
    q, table, lens = s["q"], s["table"].long(), s["lens"].long()
    seqs, heads, kv, head = lens.shape[0], case["heads"], case["kv_heads"], case["head"]
    group, tokens = heads // kv, table.shape[1] * case["page"]
    runs, starts = s["longest"], s["cum"][:-1].long()
    count = s["cum"][1:].long() - starts
    at = torch.arange(runs, device=q.device)
    token = torch.arange(tokens, device=q.device)

    def gathered(codes, scales):  # [seqs, KV heads, tokens, head]
        x = _values(codes[table], scales[table])
        return x.transpose(1, 2).reshape(seqs, kv, tokens, head)

    k, v = gathered(s["k_codes"], s["k_scales"]), gathered(s["v_codes"], s["v_scales"])
    v = torch.where((token[None, :] < lens[:, None])[:, None, :, None], v, 0.0)
    rows = (starts[:, None] + at).clamp(max=q.shape[0] - 1)
    x = q[rows].float().reshape(seqs, runs, kv, group, head).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(x.reshape(seqs, kv, group * runs, head), k.transpose(-1, -2)).mul_(s["scale"])
    del k
    scores = scores.view(seqs, kv, group, runs, tokens)
    last = (lens - count)[:, None] + at  # the last token that each new token sees
    away = token - last[..., None]       # [seqs, runs, tokens]
    if s["alibi"] is not None:
        scores += s["alibi"].view(1, kv, group, 1, 1) * away[:, None, None].float()
    scores.masked_fill_((away > 0)[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    scores /= scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(seqs, kv, group * runs, tokens), v)
    out = out.view(seqs, kv, group, runs, head).permute(0, 3, 1, 2, 4).reshape(seqs, runs, heads, head)
    row = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(s["cum"].long(), row, right=True) - 1
    return out[seq, row - starts[seq]].to(q.dtype)


# ---- the calls ----

_ops = None


def _calls():
    global _ops
    if _ops is None:
        from infinicore_amd import ops as _ops
    return _ops


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        if op == "write_read":
            _write(s)
        return _read(s) if op in ("write_read", "read") else _attention(s)
    call = _calls()
    pool = (s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"])
    if op == "write_read":
        call.paged_caching_fp4(*pool, s["k"], s["v"], s["slots"])
    if op in ("write_read", "read"):
        return call.paged_reading_fp4(*pool, s["slots"], dtype=s["dtype"])
    if op == "decode":
        return call.paged_attention_fp4(s["q"], *pool, s["table"], s["lens"], s["alibi"], s["scale"])
    return call.paged_attention_prefill_fp4(s["q"], *pool, s["table"], s["lens"], s["cum"], s["alibi"], s["scale"])


# ---- inputs ----

def _pool(case, blocks, gen, dev):
    """A pool of normal values whose channels differ in size, a few of them by a lot, as keys' do."""
    kv, page, head = case["kv_heads"], case["page"], case["head"]
    made = []
    for _ in range(2):
        size = torch.exp(0.5 * torch.randn((kv, 1, head), device=dev, generator=gen))
        size = torch.where(torch.rand((kv, 1, head), device=dev, generator=gen) < 0.02, 6 * size, size)
        codes = torch.empty((blocks, kv, page, head // 2), dtype=torch.uint8, device=dev)
        scales = torch.empty((blocks, kv, page, head // _GROUP), dtype=torch.uint8, device=dev)
        step = max(1, (1 << 25) // (kv * page * head))
        for b in range(0, blocks, step):
            n = min(step, blocks - b)
            x = torch.randn((n, kv, page, head), device=dev, generator=gen) * size
            codes[b:b + n], scales[b:b + n] = _quantised(x)
        made += [codes, scales]
    return dict(k_codes=made[0], k_scales=made[1], v_codes=made[2], v_scales=made[3])


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    dtype, kv, head, page = _DTYPES[case["dtype"]], case["kv_heads"], case["head"], case["page"]
    state = {"case": case, "dtype": dtype}
    if case["op"] in ("write_read", "read"):
        n = case["tokens"]
        blocks = -(-(2 if case["op"] == "write_read" else 1) * n // page) + 8
        if case["op"] == "write_read":
            slots = torch.randperm(blocks * page, device=dev, generator=gen)[:n]
            state["k"] = torch.randn((n, kv, head), dtype=dtype, device=dev, generator=gen)
            state["v"] = torch.randn((n, kv, head), dtype=dtype, device=dev, generator=gen)
        else:  # a sequence: the tokens of whole pages, the pages in any order
            pages = torch.randperm(blocks, device=dev, generator=gen)[:-(-n // page)]
            slots = (pages[:, None] * page + torch.arange(page, device=dev)).flatten()[:n]
        slots[torch.randperm(n, device=dev, generator=gen)[:_padding_tokens(case)]] = -1
        state.update(_pool(case, blocks, gen, dev), slots=slots)
        return state
    index = _INDEX[case["index"]]
    new, total = _lengths(case)
    order = random.Random(int(seed)).sample(range(len(new)), len(new))
    new, total = [new[i] for i in order], [total[i] for i in order]
    needed = [-(-t // page) for t in total]
    blocks = int(math.ceil(sum(needed) * (1.0 + _SPARE_PAGES)))
    pages = torch.randperm(blocks, generator=torch.Generator().manual_seed(int(seed)))
    table = torch.zeros((len(new), max(needed)), dtype=index)
    at = 0
    for s, count in enumerate(needed):
        table[s, :count] = pages[at:at + count].to(index)
        at += count
    cum = [0]
    for n in new:
        cum.append(cum[-1] + n)
    state.update(_pool(case, blocks, gen, dev), scale=1.0 / math.sqrt(head), table=table.to(dev), longest=max(new),
                 lens=torch.tensor(total, dtype=index, device=dev), cum=torch.tensor(cum, dtype=index, device=dev), alibi=None,
                 q=torch.randn((sum(new), case["heads"], head), dtype=dtype, device=dev, generator=gen))
    if case["alibi"]:
        state["alibi"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / case["heads"]) for h in range(case["heads"])], device=dev)
    return state


# ---- the same in 64 bits, from the definition ----

def _exact_rounded(x):
    """x [.., n] as the pool holds it: each group scaled by its exponent, each element the nearest of the magnitudes."""
    g = x.double().unflatten(-1, (-1, _GROUP))
    top = g.abs().amax(-1, keepdim=True)
    unit = torch.pow(2.0, (torch.frexp(top).exponent.double() - 1 - 2).clamp(-23, 13))
    m = torch.tensor(_MAGNITUDES, dtype=torch.float64, device=x.device)
    a = (g.abs() / unit).clamp(max=6.0)
    below = ((a[..., None] >= m).sum(-1) - 1).clamp(max=6)
    down, up = a - m[below], m[below + 1] - a
    code = below + ((up < down) | ((up == down) & (below % 2 == 1))).long()
    value = torch.where(torch.isfinite(top), torch.copysign(m[code] * unit, g), math.nan)
    return value.flatten(-2)


def _exact_values(codes, scales):
    c = torch.stack((codes % 16, codes // 16), dim=-1).flatten(-2).long()
    exponent, mantissa = (c >> 1) & 3, (c & 1).double()
    m = torch.where(exponent > 0, (1 + mantissa / 2) * torch.pow(2.0, exponent.double() - 1), mantissa / 2)
    unit = torch.pow(2.0, scales.double() - 127).masked_fill(scales == 255, math.nan)
    return (1 - 2 * (c >> 3)).double() * m * unit.repeat_interleave(_GROUP, dim=-1)


def exact(case, seed):
    s = prepare(case, seed)
    block = case["page"]
    if case["op"] in ("write_read", "read"):
        held = (s["slots"] >= 0).nonzero()[:, 0]
        page, row = s["slots"][held] // block, s["slots"][held] % block
        outs = []
        for name in ("k", "v"):
            out = torch.zeros((case["tokens"], case["kv_heads"], case["head"]), dtype=torch.float64, device=held.device)
            for part in held.split(8192):
                p, r = s["slots"][part] // block, s["slots"][part] % block
                out[part] = (_exact_rounded(s[name][part]) if case["op"] == "write_read"
                             else _exact_values(s[name + "_codes"][p, :, r], s[name + "_scales"][p, :, r]))
            outs.append(out)
        return tuple(outs)
    lens, cum = s["lens"].tolist(), s["cum"].tolist()
    kv, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for i, total in enumerate(lens):
        pages = s["table"][i, :-(-total // block)].long()
        n = cum[i + 1] - cum[i]
        last = torch.arange(total - n, total, device=out.device)
        away = torch.arange(total, device=out.device)[None, :] - last[:, None]
        for g in range(kv):
            k, v = (_exact_values(s[x + "_codes"][pages, g].flatten(0, 1)[:total], s[x + "_scales"][pages, g].flatten(0, 1)[:total])
                    for x in "kv")
            for h in range(g * group, (g + 1) * group):
                scores = (s["q"][cum[i]:cum[i + 1], h].double() @ k.T) * s["scale"]
                if s["alibi"] is not None:
                    scores = scores + s["alibi"][h].double() * away
                scores.masked_fill_(away > 0, -math.inf)
                out[cum[i]:cum[i + 1], h] = torch.softmax(scores, dim=-1) @ v
    return out
