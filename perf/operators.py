"""Cases for the operators that fill a paged cache and attend over it with many query tokens:

  append   rope_append_paged / rope_append_reference_paged: the new tokens of a batch (packed, one or many per
           sequence) rotated at their positions and stored in their sequences' pages, coded or bf16
  attend   attention_prefill: causal attention of packed prompts with grouped heads
  chunk    attention_prefill_paged / attention_prefill_reference_paged: the same with the keys and values in pages,
           for a prompt that continues what is cached, or for drafted tokens that are checked at once

A case names the batch by ranges; the ragged lengths inside a range follow from the case alone (see _lengths), so
work() can count them. The coded cache is lossless: its bytes are whole numbers that the plain form reproduces, so
they are returned as they are held. Only `run` goes by `own`.
"""
import math
import random

import torch

own = False

D, PAGE = 128, 16
SCALE = D ** -0.5
EPS = 1e-6


# ----------------------------------------------------------------------------- cases

def listed():
    return [
        # one decode step of a batch: every sequence's next token into its page
        dict(name="append step bf16", op="append", pool="bf16", seqs=64, new_lo=1, new_hi=1, ctx_lo=200, ctx_hi=4000,
             hq=32, hkv=8, norm=False),
        # prompts of different lengths entering a bf16 pool at once, some on a cached prefix; heads normalised first
        dict(name="append prompts bf16", op="append", pool="bf16", seqs=9, new_lo=300, new_hi=2100, ctx_lo=0,
             ctx_hi=700, hq=32, hkv=8, norm=True),
        # the decode step of the coded cache: most tokens join an open page, a sixteenth of the pages fill and are coded
        dict(name="append step coded", op="append", pool="coded", seqs=32, new_lo=1, new_hi=1, ctx_lo=900, ctx_hi=4000,
             hq=32, hkv=8, norm=False),
        # prompts entering the coded cache, starting and ending inside pages
        dict(name="append prompts coded", op="append", pool="coded", seqs=12, new_lo=100, new_hi=1500, ctx_lo=0,
             ctx_hi=400, hq=28, hkv=4, norm=False),
        # a few very short prompts: the latency of a small call
        dict(name="attend short", op="attend", seqs=3, new_lo=1, new_hi=40, ctx_lo=0, ctx_hi=0, hq=8, hkv=2),
        # one prompt of ordinary length
        dict(name="attend 4096", op="attend", seqs=1, new_lo=4096, new_hi=4096, ctx_lo=0, ctx_hi=0, hq=32, hkv=8),
        # a batch of ragged prompts, seven query heads to a KV head
        dict(name="attend ragged", op="attend", seqs=16, new_lo=33, new_hi=2047, ctx_lo=0, ctx_hi=0, hq=28, hkv=4),
        # a long prompt
        dict(name="attend 16384", op="attend", seqs=1, new_lo=16384, new_hi=16384, ctx_lo=0, ctx_hi=0, hq=32, hkv=8),
        # chunks of several prompts on top of what a bf16 pool holds of them
        dict(name="chunk bf16", op="chunk", pool="bf16", seqs=4, new_lo=100, new_hi=512, ctx_lo=1500, ctx_hi=8000,
             hq=32, hkv=8),
        # few rows on a long context: the last chunk of a long prompt
        dict(name="chunk bf16 long", op="chunk", pool="bf16", seqs=1, new_lo=61, new_hi=61, ctx_lo=32000, ctx_hi=32000,
             hq=32, hkv=8),
        # a large chunk of a long prompt over the coded cache
        dict(name="chunk coded long", op="chunk", pool="coded", seqs=1, new_lo=2048, new_hi=2048, ctx_lo=30720,
             ctx_hi=30720, hq=28, hkv=4),
        # drafted tokens of a batch checked at once over the coded cache
        dict(name="chunk coded drafts", op="chunk", pool="coded", seqs=16, new_lo=2, new_hi=8, ctx_lo=1000, ctx_hi=4000,
             hq=32, hkv=8),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    hq, hkv = rng.choice([(32, 8), (28, 4), (16, 8), (8, 2), (40, 8), (12, 4), (8, 8), (64, 4), (16, 1)])
    op = rng.choice(["append", "attend", "chunk"])
    if op == "append":
        pool = rng.choice(["bf16", "coded"])
        seqs = _spread(rng, 1, 96)
        lo = rng.choice([1, _spread(rng, 1, 64)])
        hi = max(lo, _spread(rng, 1, max(1, 16384 // seqs))) if rng.random() < 0.6 else lo
        ctx = _spread(rng, 1, 4000)
        return dict(op=op, pool=pool, seqs=seqs, new_lo=lo, new_hi=hi, ctx_lo=rng.choice([0, ctx // 3]), ctx_hi=ctx,
                    hq=hq, hkv=hkv, norm=pool == "bf16" and rng.random() < 0.5)
    if op == "attend":
        hi = _spread(rng, 1, 8192)
        seqs = _spread(rng, 1, max(1, min(32, 32768 // hi)))
        return dict(op=op, seqs=seqs, new_lo=_spread(rng, 1, hi), new_hi=hi, ctx_lo=0, ctx_hi=0, hq=hq, hkv=hkv)
    ctx = _spread(rng, 16, 32000)
    seqs = _spread(rng, 1, max(1, min(32, 64000 // ctx)))
    hi = _spread(rng, 1, max(1, min(2048, 8192 // seqs)))
    return dict(op=op, pool=rng.choice(["bf16", "coded"]), seqs=seqs, new_lo=_spread(rng, 1, hi), new_hi=hi,
                ctx_lo=_spread(rng, 1, ctx), ctx_hi=ctx, hq=hq, hkv=hkv)


def _lengths(case):
    """New tokens of each sequence and the tokens it held before: spread over their ranges by the golden ratio."""
    def within(lo, hi, b, phase):
        return lo + int((hi - lo + 1) * ((b * 0.6180339887 + phase) % 1.0))

    if case["seqs"] == 1:
        return [case["new_hi"]], [case["ctx_hi"]]
    seqs = range(case["seqs"])
    new = [within(case["new_lo"], case["new_hi"], b, 0.93) for b in seqs]
    return new, [within(case["ctx_lo"], case["ctx_hi"], b, 0.31) for b in seqs]


def work(case):
    new, ctx = _lengths(case)
    hq, hkv = case["hq"], case["hkv"]
    n, rows = sum(new), sum(new) + sum(ctx)
    q_bytes, kv_bytes = n * hq * D * 2, n * hkv * D * 2
    if case["op"] == "append":
        if case["pool"] == "bf16":
            stored = 2 * kv_bytes
        else:  # whole pages are read from and written as coded rows; what stays open is stored raw
            done = sum((c + m) // PAGE * PAGE - c // PAGE * PAGE for m, c in zip(new, ctx))
            left = sum(min(m, (c + m) % PAGE) for m, c in zip(new, ctx))
            early = sum(c % PAGE for m, c in zip(new, ctx) if c % PAGE and (c + m) // PAGE > c // PAGE)
            stored = 2 * hkv * (done * (128 + 64 + 8) + (left + early) * 256)
        flops = n * (hq + hkv) * D * (3 + (3 if case["norm"] else 0))
        return {"bytes": 2 * q_bytes + 2 * kv_bytes + stored + n * D * 4, "flops": flops}
    pairs = sum(m * c + m * (m + 1) // 2 for m, c in zip(new, ctx))
    if case["op"] == "attend":
        held = 2 * kv_bytes
    elif case["pool"] == "bf16":
        held = 2 * rows * hkv * D * 2
    else:
        held = int(2 * rows * hkv * 200.5)
    return {"bytes": 2 * q_bytes + held, "flops": 4 * D * hq * pairs}


# ----------------------------------------------------------------------------- inputs

def _values(g, rows, heads, scales, zeros):
    """bf16 rows of a cache: channels of different magnitude, a few exact zeros, a few rows with a far smaller value."""
    dev = scales.device
    x = torch.randn(rows, heads, D, generator=g, device=dev) * scales
    if zeros:
        x.masked_fill_(torch.rand(rows, heads, D, generator=g, device=dev) < 4e-4, 0.0)
    odd = torch.rand(rows, heads, 1, generator=g, device=dev) < 3e-3
    channel = torch.randint(0, D, (rows, heads, 1), generator=g, device=dev)
    hit = odd & (torch.arange(D, device=dev) == channel)
    return torch.where(hit, x * 2.0 ** -20, x).to(torch.bfloat16)


def _inputs(case, seed):
    """Everything that the seed decides, before it is laid out: also what exact() starts from."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    new, ctx = _lengths(case)
    hq, hkv, n, held = case["hq"], case["hkv"], sum(new), sum(ctx)
    scale = lambda: torch.exp2(torch.randint(-4, 4, (hkv, D), generator=g, device="cuda").float())  # noqa: E731
    k_scale, v_scale = scale(), scale()
    x = dict(new=new, ctx=ctx, q=torch.randn(n, hq, D, generator=g, device="cuda").to(torch.bfloat16),
             k=_values(g, n, hkv, k_scale, True), v=_values(g, n, hkv, v_scale, False),
             k_held=_values(g, held, hkv, k_scale, True), v_held=_values(g, held, hkv, v_scale, False))
    if case["op"] == "append":
        angle = torch.arange(max(a + b for a, b in zip(new, ctx)), device="cuda", dtype=torch.float64)[:, None] * (
            5e5 ** (-torch.arange(64, device="cuda", dtype=torch.float64) / 64))
        x["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        if case["norm"]:
            x["q_norm"] = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(torch.bfloat16)
            x["k_norm"] = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(torch.bfloat16)
    if case["op"] != "attend":
        pages = [-(-(a + b) // PAGE) for a, b in zip(new, ctx)]
        spare = 3 + sum(pages) // 8
        order = torch.randperm(sum(pages) + spare, generator=g, device="cuda").int()
        table = torch.full((len(pages), max(pages)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, m in enumerate(pages):
            table[b, :m] = order[at:at + m]
            at += m
        x["block_table"], x["pool_pages"] = table, sum(pages) + spare
    return x


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(lengths):
    at = [0]
    for m in lengths:
        at.append(at[-1] + m)
    return _ints(at)


def _places(lengths, first, device="cuda"):
    """Sequence and position of each of a batch's packed tokens."""
    m = torch.tensor(lengths, device=device)
    seq = torch.repeat_interleave(torch.arange(len(lengths), device=device), m)
    at = torch.arange(len(seq), device=device) - (torch.cumsum(m, 0) - m)[seq]
    return seq, at + torch.tensor(first, device=device)[seq]


def prepare(case, seed):
    x = _inputs(case, seed)
    new, ctx = x["new"], x["ctx"]
    s = dict(op=case["op"], pool=case.get("pool"), q=x["q"], k=x["k"], v=x["v"], cu_seqlens=_starts(new))
    if case["op"] == "attend":
        return s
    hkv = case["hkv"]
    s.update(block_table=x["block_table"], seq_lens=_ints([a + b for a, b in zip(new, ctx)]))
    if case["op"] == "append":
        s.update(cos_sin=x["cos_sin"], q_norm=x.get("q_norm"), k_norm=x.get("k_norm"),
                 one_each=all(m == 1 for m in new))
        lengths, rows = ctx, {"k": x["k_held"], "v": x["v_held"]}
    else:  # the chunk's own keys and values are in the cache as well
        lengths = [a + b for a, b in zip(new, ctx)]
        held_seq, _ = _places(ctx, [0] * len(ctx))
        new_seq, _ = _places(new, [0] * len(new))
        back = torch.argsort(torch.cat([held_seq, new_seq]), stable=True)
        rows = {"k": torch.cat([x["k_held"], x["k"]])[back], "v": torch.cat([x["v_held"], x["v"]])[back]}
    seq, pos = _places(lengths, [0] * len(lengths))
    for name in ("k", "v"):
        if case["pool"] == "bf16":
            pool = torch.zeros(1, x["pool_pages"] * PAGE, hkv, D, dtype=torch.bfloat16, device="cuda")
            pool[0, _row_of(s["block_table"], seq, pos)] = rows[name]
        else:
            pool = _empty_coded(x["pool_pages"], hkv, len(new), 512 + (len(seq) + len(s["k"])) * hkv // 4)
            _append_coded(pool, rows[name], seq, pos, s["block_table"], _ints(lengths))
        s[name + "_pool"] = pool
    return s


def _empty_coded(pages, heads, seqs, cap):
    """An empty coded pool: `cap` raw slots, then one open page of 16 rows per (sequence, head)."""
    byte = dict(dtype=torch.uint8, device="cuda")
    word = dict(dtype=torch.int32, device="cuda")
    return dict(shape=(1, pages * PAGE, heads, D), sm=torch.zeros(1, pages * PAGE, heads, D, **byte),
                code=torch.zeros(1, pages * PAGE, heads, D // 2, **byte),
                base=torch.zeros(1, pages, heads, D, **byte), rowmask=torch.zeros(1, pages, heads, **word),
                rowoff=torch.zeros(1, pages, heads, **word),
                raw=torch.zeros(cap + seqs * heads * PAGE, D, dtype=torch.bfloat16, device="cuda"),
                cnt=torch.zeros(1, **word), cap=cap)


# ----------------------------------------------------------------------------- one pass

def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "append":
        return _plain_append(s)
    if s["op"] == "attend":
        return _plain_attention(s["q"], s["k"], s["v"], s["cu_seqlens"], s["cu_seqlens"])
    if s["pool"] == "bf16":
        k, v = (s[name].view(-1, s[name].shape[2], D) for name in ("k_pool", "v_pool"))
    else:
        k, v = _decode(s["k_pool"]), _decode(s["v_pool"])
    lens = s["seq_lens"].long()
    cu = torch.cat([lens.new_zeros(1), lens.cumsum(0)])
    seq, pos = _packed(cu, int(cu[-1]), lens.new_zeros(len(lens)))
    rows = _row_of(s["block_table"], seq, pos)
    return _plain_attention(s["q"], k[rows], v[rows], s["cu_seqlens"], cu)


def _run_own(s):
    from exactkv_b200 import kernels
    if s["op"] == "append":
        call = kernels.rope_append_paged if s["pool"] == "coded" else kernels.rope_append_reference_paged
        q = call(s["q"], s["k"], s["v"], s["cos_sin"], s["k_pool"], s["v_pool"], s["block_table"], s["seq_lens"],
                 cu_seqlens=None if s["one_each"] else s["cu_seqlens"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
        return dict(q=q, k=_buffers(s["k_pool"]), v=_buffers(s["v_pool"]))
    if s["op"] == "attend":
        return kernels.attention_prefill(s["q"], s["k"], s["v"], s["cu_seqlens"])
    call = kernels.attention_prefill_paged if s["pool"] == "coded" else kernels.attention_prefill_reference_paged
    return call(s["q"], s["k_pool"], s["v_pool"], s["block_table"], s["seq_lens"], s["cu_seqlens"])


_FIELDS = ("sm", "code", "base", "rowmask", "rowoff", "raw", "cnt")


def _buffers(pool):
    return {f: pool[f] for f in _FIELDS} if isinstance(pool, dict) else pool


# ----------------------------------------------------------------------------- the plain forms

def _packed(cu, n, first):
    """Sequence and position of packed tokens 0 .. n - 1; sequence b starts at position first[b]."""
    at = torch.arange(n, device=cu.device)
    seq = (at[:, None] >= cu[None, 1:]).sum(1)
    return seq, at - cu[seq] + first[seq]


def _row_of(table, seq, pos):
    return table[seq, pos // PAGE].long() * PAGE + pos % PAGE


def _rotate(x, cos_sin, weight):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    c, s = cos_sin[:, None, :64], cos_sin[:, None, 64:]
    lo, hi = x[..., :64], x[..., 64:]
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1).to(torch.bfloat16)


def _plain_append(s):
    cu, lens = s["cu_seqlens"].long(), s["seq_lens"].long()
    seq, pos = _packed(cu, s["q"].shape[0], lens - (cu[1:] - cu[:-1]))
    cs = s["cos_sin"][pos]
    q, k = _rotate(s["q"], cs, s["q_norm"]), _rotate(s["k"], cs, s["k_norm"])
    if s["pool"] == "bf16":
        rows = _row_of(s["block_table"], seq, pos)
        s["k_pool"][0, rows], s["v_pool"][0, rows] = k, s["v"]
    else:
        _append_coded(s["k_pool"], k, seq, pos, s["block_table"], s["seq_lens"])
        _append_coded(s["v_pool"], s["v"], seq, pos, s["block_table"], s["seq_lens"])
    return dict(q=q, k=_buffers(s["k_pool"]), v=_buffers(s["v_pool"]))


def _append_coded(c, x, seq, pos, table, lens):
    """Rows x of (seq, pos) into the coded pool c: pages that they complete are coded, the others stay open."""
    if not len(x):
        return
    heads, cap, wide = c["shape"][2], c["cap"], table.shape[1]
    lens = lens.long()
    touched, which = torch.unique(seq * wide + pos // PAGE, return_inverse=True)
    b, pg = touched // wide, touched % wide
    tails = c["raw"][cap:].view(-1, heads, PAGE, D)
    rows = tails[b].clone()                                          # [U, H, 16, D]: what the open pages hold
    rows[which, :, pos % PAGE] = x
    page = table[b, pg].long()
    full = (pg + 1) * PAGE <= lens[b]

    u = rows[full].view(torch.int16).int() & 0xFFFF                  # the complete pages' bits [F, H, 16, D]
    e = u >> 7 & 0xFF
    low = (e.amax(2, keepdim=True) - 15).clamp(min=0)                # first exponent of the channel's window
    zero = ((e == 0).any(2, keepdim=True) & (low > 0)).int()         # a zero that the window does not reach
    raw = (((e < low + zero) & (e != 0)) | (low >= 128)).any(-1)     # rows kept as they are [F, H, 16]
    code = (e - low).clamp(0, 15)
    at = page[full]
    c["sm"].view(-1, PAGE, heads, D)[at] = (u >> 8 & 0x80 | u & 0x7F).to(torch.uint8).transpose(1, 2)
    c["code"].view(-1, PAGE, heads, D // 2)[at] = (code[..., :64] | code[..., 64:] << 4).to(torch.uint8).transpose(1, 2)
    c["base"][0, at] = (low + 128 * zero).clamp(max=255)[:, :, 0].to(torch.uint8)
    c["rowmask"][0, at] = (raw.int() << torch.arange(PAGE, device=x.device, dtype=torch.int32)).sum(-1).int()
    count = raw.sum(-1)
    end = count.flatten().cumsum(0).view_as(count) + c["cnt"]
    c["rowoff"][0, at] = (end - count).int()
    slot = (end - count)[..., None] + raw.cumsum(-1) - raw.long()
    keep = raw & (slot < cap)
    c["raw"][slot[keep]] = rows[full][keep]
    c["cnt"] += raw.sum().int()

    still = ~full
    tails[b[still]] = rows[still]
    c["rowmask"][0, page[still]] = (1 << PAGE) - 1
    first = cap + PAGE * (b[still, None] * heads + torch.arange(heads, device=x.device))
    c["rowoff"][0, page[still]] = first.int()


def _decode(c):
    """All rows that a coded pool holds, as bf16 [rows, heads, 128]."""
    heads = c["shape"][2]
    code = c["code"].view(-1, PAGE, heads, D // 2).int()
    code = torch.cat([code & 15, code >> 4], -1)
    base = c["base"].view(-1, 1, heads, D).int()
    e = torch.where((base >= 128) & (code == 0), 0, (base & 127) + code)
    s = c["sm"].view(-1, PAGE, heads, D).int()
    x = ((s & 0x80) << 8 | e << 7 | s & 0x7F).to(torch.int16).view(torch.bfloat16)
    raw = (c["rowmask"].view(-1, 1, heads) >> torch.arange(PAGE, device=x.device)[:, None] & 1).bool()
    slot = c["rowoff"].view(-1, 1, heads) + raw.cumsum(1) - raw.long()
    return torch.where(raw[..., None], c["raw"][slot.clamp(0, len(c["raw"]) - 1)], x).view(-1, heads, D)


def _plain_attention(q, k, v, cu_q, cu_k):
    """Causal attention of packed queries over packed keys, the last query of a sequence at its last key."""
    hq, hkv = q.shape[1], k.shape[1]
    cu_q, cu_k = cu_q.long(), cu_k.long()
    nq, nk = cu_q[1:] - cu_q[:-1], cu_k[1:] - cu_k[:-1]
    mq, mk = int(nq.max()), int(nk.max())
    i, j = torch.arange(mq, device=q.device), torch.arange(mk, device=q.device)
    iq = (cu_q[:-1, None] + i).clamp(max=len(q) - 1)                  # [B, mq] padded
    jk = (cu_k[:-1, None] + j).clamp(max=len(k) - 1)
    last = i[None] + (nk - nq)[:, None]                               # the last key that each query sees
    sees = (j[None, None] <= last[..., None]) & (j < nk[:, None])[:, None]
    out = torch.empty(len(nq), mq, hq, D, dtype=q.dtype, device=q.device)
    g = hq // hkv
    for h in range(hkv):  # a KV head at a time: the scores of all heads need not exist at once
        qh = q[iq, h * g:(h + 1) * g].float().transpose(1, 2)         # [B, g, mq, D]
        s = qh @ k[jk, h].float().transpose(1, 2)[:, None] * SCALE
        s = s.masked_fill(~sees[:, None], -math.inf)
        m = s.amax(-1, keepdim=True).clamp(min=-1e30)
        p = (s - m).exp()
        del s
        o = p @ v[jk, h].float()[:, None] / p.sum(-1, keepdim=True).clamp(min=1e-30)
        out[:, :, h * g:(h + 1) * g] = o.transpose(1, 2).to(q.dtype)
    seq, at = _packed(cu_q, len(q), torch.zeros_like(nq))
    return out[seq, at]


# ----------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    x = _inputs(case, seed)
    new, ctx = x["new"], x["ctx"]
    if case["op"] == "append":
        return _exact_append(case, x)
    g = case["hq"] // case["hkv"]
    out, at_q, at_k = [], 0, 0
    for m, c in zip(new, ctx):
        q = x["q"][at_q:at_q + m].double()
        k = torch.cat([x["k_held"][at_k:at_k + c], x["k"][at_q:at_q + m]]).double()
        v = torch.cat([x["v_held"][at_k:at_k + c], x["v"][at_q:at_q + m]]).double()
        o = torch.empty(m, case["hq"], D, dtype=torch.float64, device="cuda")
        for h in range(case["hq"]):
            for i in range(0, m, 4096):
                r = range(i, min(m, i + 4096))
                z = torch.mm(q[i:r.stop, h], k[:c + r.stop, h // g].T) / math.sqrt(D)
                z += torch.triu(torch.full_like(z, -math.inf), diagonal=c + i + 1)
                o[i:r.stop, h] = torch.mm(torch.softmax(z, 1), v[:c + r.stop, h // g])
        out.append(o)
        at_q, at_k = at_q + m, at_k + c
    return torch.cat(out)


def _exact_append(case, x):
    """The rotation as a product of complex numbers, a sequence at a time."""
    half = D // 2
    outs, at = {"q": [], "k": []}, 0
    pools = {n: torch.zeros(1, x["pool_pages"] * PAGE, case["hkv"], D, dtype=torch.float64, device="cuda")
             for n in ("k", "v")}
    held = 0
    for b, (m, c) in enumerate(zip(x["new"], x["ctx"])):
        turn = x["cos_sin"][c:c + m].double()
        turn = torch.complex(turn[:, :half], turn[:, half:])[:, None]
        for name in outs:
            y = x[name][at:at + m].double()
            if case["norm"]:
                y = x[name + "_norm"].double() * y / ((y * y).sum(-1, keepdim=True) / D + EPS).sqrt()
            y = torch.complex(y[..., :half].contiguous(), y[..., half:].contiguous()) * turn
            outs[name].append(torch.cat([y.real, y.imag], -1))
        if case["pool"] == "bf16":
            rows = x["block_table"][b].long()[:, None] * PAGE + torch.arange(PAGE, device="cuda")
            rows = rows.flatten()[:c + m]
            pools["k"][0, rows] = torch.cat([x["k_held"][held:held + c].double(), outs["k"][-1]])
            pools["v"][0, rows] = torch.cat([x["v_held"][held:held + c], x["v"][at:at + m]]).double()
        at, held = at + m, held + c
    if case["pool"] == "bf16":
        return dict(q=torch.cat(outs["q"]), **pools)
    return dict(q=torch.cat(outs["q"]), k=None, v=None)
