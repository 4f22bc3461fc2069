"""New tokens into paged caches (exk_rope_append_bf16, exk_rope_append_compressed).

The rotation is defined to the bit (fp32 products and sums rounded one by one,
one rounding to bf16), so without the norm queries, bf16 pools and the
compressed bytes are compared for equality: the compressed pages with the
oracle's encoder. With the norm the bound is, per channel,
    2^-8 |y| + 2^-18 (|a| + |b|)
for y = a + b or a - b of the rotated pair: one rounding to bf16 (half a step) and
fp32 arithmetic before it (a sum of 128 squares, rsqrt, four products: fewer than
64 roundings of 2^-24 each).
"""
import numpy as np
import pytest
import torch

import exactkv_b200 as ekv
from exactkv_b200 import kernels, synthetic
from gpu_util import same_bits, to_bits
from oracle import codec as ocodec

D = 128
THETA = 1e6


def offsets(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def table_of(n, device="cuda"):
    inv = THETA ** (-torch.arange(64, dtype=torch.float64, device=device) / 64)
    return ekv.rope_table(inv, n)


def rotated(x, cs, w=None, eps=1e-6):
    """The definition on the CPU: x [n, H, 128] bf16, cs [n, 128] fp32. Without w in
    fp32 step by step (exact bits); with w in fp64: (y, tolerance)."""
    x, cs = x.cpu().float().numpy(), cs.cpu().numpy()
    c, s = cs[:, None, :64], cs[:, None, 64:]
    if w is None:
        lo, hi = x[..., :64], x[..., 64:]
        y = np.concatenate([lo * c - hi * s, hi * c + lo * s], -1)
        return torch.from_numpy(y).to(torch.bfloat16)
    x = x.astype(np.float64)
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.double().cpu().numpy()
    lo, hi = x[..., :64], x[..., 64:]
    a, b = np.concatenate([lo * c, hi * c], -1), np.concatenate([-hi * s, lo * s], -1)
    y = a + b
    return torch.from_numpy(y), torch.from_numpy(2.0 ** -8 * np.abs(y) + 2.0 ** -18 * (np.abs(a) + np.abs(b)))


def tokens(n, Hq, Hkv, seed):
    q = synthetic.make_q(n, Hq, seed=seed) if n else torch.zeros(0, Hq, D, dtype=torch.bfloat16, device="cuda")
    if not n:
        return q, *(torch.zeros(0, Hkv, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    k = synthetic.make_kv(1, n, Hkv, seed=seed + 1, key=True, raw_frac=0.02)[0]
    v = synthetic.make_kv(1, n, Hkv, seed=seed + 2, key=False, raw_frac=0.02)[0]
    return q, k, v


class Model:
    """What the sequences should hold: their rotated keys and values by position."""

    def __init__(self, B, Hkv, max_pages, spare=3, seed=0, tails=None):
        self.B, self.H, self.max_pages = B, Hkv, max_pages
        self.pages = B * max_pages + spare
        perm = torch.randperm(self.pages, generator=torch.Generator().manual_seed(seed)).int()
        self.table = perm[:B * max_pages].view(B, max_pages).cuda()
        self.k = [torch.zeros(0, Hkv, D, dtype=torch.bfloat16) for _ in range(B)]
        self.v = [torch.zeros(0, Hkv, D, dtype=torch.bfloat16) for _ in range(B)]
        self.kb, self.vb = (torch.zeros(1, self.pages * 16, Hkv, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.kc, self.vc = (ekv.PagedCompressedKV(self.pages, Hkv, D, tails or B, reserve=1.0) for _ in range(2))
        self.cs = table_of(max_pages * 16)
        self.raw_rows = [0, 0]

    def lens(self):
        return [len(k) for k in self.k]

    def append(self, new, Hq, seed, packed=True, slots=None, pad=0):
        q, k, v = tokens(sum(new) + pad, Hq, self.H, seed)
        start = self.lens()
        a = 0
        want_q = []
        for b, n in enumerate(new):
            cs = self.cs[start[b]:start[b] + n]
            want_q.append(rotated(q[a:a + n], cs))
            self.k[b] = torch.cat([self.k[b], rotated(k[a:a + n], cs)])
            self.v[b] = torch.cat([self.v[b], v[a:a + n].cpu()])
            self._count(b, start[b], start[b] + n)
            a += n
        sl = ints(self.lens())
        cu = offsets(new) if packed else None
        out = torch.full_like(q, 5.0)
        got = ekv.rope_append_reference_paged(q, k, v, self.cs, self.kb, self.vb, self.table, sl, cu, q_out=out)
        assert got is out and same_bits(out[:a].cpu(), torch.cat(want_q))
        assert (out[a:] == 5).all()
        out2 = ekv.rope_append_paged(q, k, v, self.cs, self.kc, self.vc, self.table, sl, cu, slots=slots)
        assert same_bits(out2[:a], out[:a])
        kernels.check_status()

    def _count(self, b, start, end):
        """Raw rows of the pages that this append completes."""
        for i, x in enumerate((self.k[b], self.v[b])):
            lo, hi = start // 16 * 16, end // 16 * 16
            if hi > lo:
                e = ocodec.encode(to_bits(x[lo:hi])[None])
                self.raw_rows[i] += len(e["raw"])

    def check(self, slots=None):
        for i, (xs, bf, c) in enumerate(((self.k, self.kb, self.kc), (self.v, self.vb, self.vc))):
            assert int(c.cnt.item()) == self.raw_rows[i]
            pool = bf.view(self.pages, 16, self.H, D).cpu()
            for b, x in enumerate(xs):
                n = len(x)
                if n == 0:
                    continue
                pg = self.table[b, :-(-n // 16)].long().cpu()
                assert same_bits(pool[pg].reshape(-1, self.H, D)[:n], x)
                full = n // 16
                if full:
                    e = ocodec.encode(to_bits(x[:full * 16])[None])
                    f = pg[:full]
                    for name in ("sm", "code"):
                        got = getattr(c, name).view(self.pages, 16, self.H, -1).cpu()[f].numpy()
                        assert np.array_equal(got.reshape(e[name][0].shape), e[name][0]), name
                    for name in ("base", "rowmask"):
                        assert np.array_equal(getattr(c, name)[0].cpu()[f].numpy(), e[name][0]), name
                dec = ocodec.decode({**{m: getattr(c, m).cpu().numpy() for m in ("sm", "code", "base", "rowmask", "rowoff")},
                                     "raw": to_bits(c.raw), "shape": (1, self.pages * 16, self.H, D)})
                got = dec[0].reshape(self.pages, 16, self.H, D)[pg.numpy()].reshape(-1, self.H, D)[:n]
                assert np.array_equal(got, to_bits(x)), b
                if n % 16:
                    slot = b if slots is None else slots[b]
                    assert (c.rowmask[0, pg[-1]] == 0xFFFF).all()
                    first = c.cap + 16 * (slot * self.H + torch.arange(self.H))
                    assert torch.equal(c.rowoff[0, pg[-1]].cpu(), first.int())


STEPS = [
    [[5]],                                                    # one open page
    [[16], [16]],                                             # whole pages
    [[1], [14], [1], [1]],                                    # a page filled token by token
    [[7, 0, 33], [9, 40, 1], [1, 1, 1], [30, 3, 15]],         # pages completed and left open in one call, an empty sequence
    [[0, 0, 0, 5], [0, 12, 0, 12]],
    [[20], [13]],                                             # completes the open page (its rows in the tail), opens the next
    [[31, 17, 1], [18, 35, 46]],
    [[300, 1, 129], [77, 200, 2]],
]


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (7, 1), (28, 4), (3, 3)])
@pytest.mark.parametrize("case", range(len(STEPS)))
def test_steps_store_exactly_what_they_should(case, Hq, Hkv):
    steps = STEPS[case]
    m = Model(len(steps[0]), Hkv, 32, seed=case)
    for i, new in enumerate(steps):
        m.append(new, Hq, seed=100 * case + 10 * i, pad=3 * i)
        m.check()


@pytest.mark.gpu
def test_single_token_steps_and_moving_slots():
    """One token per sequence without cu_seqlens, with tail slots that are not the
    batch's order, over page boundaries."""
    B = 5
    slots = [6, 0, 3, 2, 5]
    m = Model(B, 2, 8, seed=4, tails=7)
    m.append([15, 1, 16, 30, 7], 8, seed=1, slots=ints(slots))
    for i in range(20):
        m.append([1] * B, 8, seed=50 + 3 * i, packed=False, slots=ints(slots))
    m.check(slots)
    assert min(m.lens()) == 21


@pytest.mark.gpu
def test_raw_slots_follow_sequence_page_head_order():
    """rowoff is the running count in (sequence, page, head) order, also over more
    page-heads than one CTA of the second kernel takes."""
    new = [700, 450, 16 * 80]
    m = Model(3, 4, 90, seed=6)
    m.append(new, 4, seed=9)
    for xs, c in ((m.k, m.kc), (m.v, m.vc)):
        at = 0
        for b, x in enumerate(xs):
            full = len(x) // 16
            e = ocodec.encode(to_bits(x[:full * 16])[None])
            got = c.rowoff[0].cpu()[m.table[b, :full].long().cpu()].numpy()
            assert np.array_equal(got, e["rowoff"][0] + at)
            at += len(e["raw"])
    m.check()


@pytest.mark.gpu
def test_many_sequences_and_rows_before_the_first():
    """70 sequences, some without new tokens, in a batch whose first rows belong to
    none: those rows and their queries are left alone."""
    B, Hq, Hkv, pad = 70, 4, 2, 5
    new = [(5 * i) % 23 for i in range(B)]
    q, k, v = tokens(sum(new) + pad, Hq, Hkv, seed=80)
    m = Model(B, Hkv, 3, seed=14)
    cu, sl = offsets(new) + pad, ints(new)
    out = [torch.full_like(q, 5.0) for _ in range(2)]
    ekv.rope_append_reference_paged(q, k, v, m.cs, m.kb, m.vb, m.table, sl, cu, q_out=out[0])
    ekv.rope_append_paged(q, k, v, m.cs, m.kc, m.vc, m.table, sl, cu, q_out=out[1])
    kernels.check_status()
    assert same_bits(*out) and (out[0][:pad] == 5).all()
    at = pad
    for b, n in enumerate(new):
        assert same_bits(out[0][at:at + n].cpu(), rotated(q[at:at + n], m.cs[:n]))
        m.k[b], m.v[b] = rotated(k[at:at + n], m.cs[:n]), v[at:at + n].cpu()
        m._count(b, 0, n)
        at += n
    m.check()


@pytest.mark.gpu
def test_appends_from_two_threads_on_one_stream():
    """Two threads append to pools of their own on one stream, their calls' launches
    interleaved as they come: each call's scratch is its own."""
    import threading
    models = [Model(3, 2, 40, seed=20 + i) for i in range(2)]
    steps = [[[200, 37, 5], [100, 300, 17], [1, 1, 1], [31, 15, 40]], [[16, 0, 90], [7, 333, 1], [40, 41, 42], [1, 2, 3]]]
    data = [[tokens(sum(new), 4, 2, seed=500 + 50 * i + 3 * j) for j, new in enumerate(s)] for i, s in enumerate(steps)]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()

    def run(i):
        m, lens = models[i], [0, 0, 0]
        with torch.cuda.stream(stream):
            for new, (q, k, v) in zip(steps[i], data[i]):
                lens = [a + b for a, b in zip(lens, new)]
                ekv.rope_append_paged(q, k, v, m.cs, m.kc, m.vc, m.table, ints(lens), offsets(new))
                ekv.rope_append_reference_paged(q, k, v, m.cs, m.kb, m.vb, m.table, ints(lens), offsets(new))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    kernels.check_status()
    for m, s, d in zip(models, steps, data):
        lens = [0, 0, 0]
        for new, (q, k, v) in zip(s, d):
            at = 0
            for b, n in enumerate(new):
                m.k[b] = torch.cat([m.k[b], rotated(k[at:at + n], m.cs[lens[b]:lens[b] + n])])
                m.v[b] = torch.cat([m.v[b], v[at:at + n].cpu()])
                m._count(b, lens[b], lens[b] + n)
                lens[b] += n
                at += n
        m.check()


@pytest.mark.gpu
def test_norm_before_the_rotation():
    Hq, Hkv, new, start = 12, 4, [40, 1, 3], [3, 15, 0]
    g = torch.Generator(device="cuda").manual_seed(1)
    wq, wk = (torch.randn(D, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    q, k, v = tokens(44, Hq, Hkv, seed=70)
    q *= 30
    cs = table_of(64)
    m = Model(3, Hkv, 4, seed=8)
    sl = ints([a + b for a, b in zip(new, start)])
    got = ekv.rope_append_reference_paged(q, k, v, cs, m.kb, m.vb, m.table, sl, offsets(new), q_norm=wq, k_norm=wk)
    out2 = ekv.rope_append_paged(q, k, v, cs, m.kc, m.vc, m.table, sl, offsets(new), q_norm=wq, k_norm=wk)
    assert same_bits(got, out2)
    pos = torch.cat([torch.arange(n) + s for n, s in zip(new, start)])
    y, tol = rotated(q, cs.cpu()[pos], wq)
    assert ((got.double().cpu() - y).abs() <= tol).all()
    y, tol = rotated(k, cs.cpu()[pos], wk)
    rows = torch.cat([m.table[b].long().cpu()[(torch.arange(n) + s) // 16] * 16 + (torch.arange(n) + s) % 16
                      for b, (n, s) in enumerate(zip(new, start))])
    assert ((m.kb[0].cpu()[rows].double() - y).abs() <= tol).all()
    assert same_bits(m.vb[0].cpu()[rows], v.cpu())
    # the open pages of the compressed pool hold the same bits (sequence 1 filled its page)
    dec = kernels.decode_to_bf16(m.kc.buffers(), m.kc.TS)[0].cpu()
    last = rows[-3:]
    assert same_bits(dec[last], m.kb[0].cpu()[last])
    kernels.check_status()


@pytest.mark.gpu
def test_strided_views_and_rotation_in_place():
    """q, k, v as views of one projection; q_out = q."""
    Hq, Hkv, n = 8, 2, 50
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn(n, Hq + 2 * Hkv, D, generator=g, device="cuda").to(torch.bfloat16)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    m = Model(1, Hkv, 4, seed=3)
    cs = m.cs
    want = rotated(q, cs[:n])
    wk, wv = rotated(k, cs[:n]), v.cpu().clone()
    held = qkv[:, Hq:].clone()
    out = ekv.rope_append_paged(q, k, v, cs, m.kc, m.vc, m.table, ints([n]), offsets([n]), q_out=q)
    assert out is q and same_bits(q.cpu(), want) and same_bits(qkv[:, Hq:], held)
    m.k, m.v = [wk], [wv]
    m.kb[0, (m.table[0, :4].long()[:, None] * 16 + torch.arange(16, device="cuda")).flatten()[:n]] = wk.cuda()
    m.vb[0, (m.table[0, :4].long()[:, None] * 16 + torch.arange(16, device="cuda")).flatten()[:n]] = wv.cuda()
    m._count(0, 0, n)
    m.check()


@pytest.mark.gpu
def test_positions_and_pages_out_of_range_are_not_stored():
    Hq, Hkv = 4, 2
    q, k, v = tokens(20, Hq, Hkv, seed=90)
    for lens in ([40, 10], [5, 10]):                  # past the block table (2 pages); before position 0
        m = Model(2, Hkv, 2, seed=5)
        sl, cu = ints(lens), offsets([10, 10])
        want = m.kb.clone()
        out = ekv.rope_append_reference_paged(q, k, v, m.cs, m.kb, m.vb, m.table, sl, cu)
        with pytest.raises(RuntimeError, match="position"):
            kernels.check_status()
        pos = torch.arange(10) + lens[0] - 10
        ok = (pos >= 0) & (pos < 32)
        assert (out[:10].cpu()[~ok] == 0).all()
        rows = m.table[0].long().cpu()[pos[ok] // 16] * 16 + pos[ok] % 16
        rows2 = m.table[1, 0].long().cpu() * 16 + torch.arange(10)
        want[0, rows.cuda()] = rotated(k[:10][ok.cuda()], m.cs.cpu()[pos[ok]]).cuda()
        want[0, rows2.cuda()] = rotated(k[10:], m.cs[:10]).cuda()
        assert same_bits(m.kb, want)
        ekv.rope_append_paged(q, k, v, m.cs, m.kc, m.vc, m.table, sl, cu)
        with pytest.raises(RuntimeError, match="position"):
            kernels.check_status()
        used = (m.kc.rowmask[0] != 0).any(1).nonzero().flatten().tolist()
        assert used == [int(m.table[1, 0])]           # the other sequence alone
    m = Model(2, Hkv, 2, seed=5)
    bad = m.table.clone()
    bad[0, 0] = m.pages
    for call, pools in ((ekv.rope_append_reference_paged, (m.kb, m.vb)), (ekv.rope_append_paged, (m.kc, m.vc))):
        out = call(q, k, v, m.cs, *pools, bad, ints([10, 10]), offsets([10, 10]))
        with pytest.raises(RuntimeError, match="outside the pool"):
            kernels.check_status()
        assert same_bits(out[:10].cpu(), rotated(q[:10], m.cs[:10]))
    assert int((m.kb != 0).any(-1).any(-1).sum()) == 10
    # a tail slot that the pool does not have; bounds that are no batch's
    ekv.rope_append_paged(q, k, v, m.cs, m.kc, m.vc, m.table, ints([10, 10]), offsets([10, 10]), slots=ints([0, 2]))
    with pytest.raises(RuntimeError, match="tail slot"):
        kernels.check_status()
    before = m.kb.clone()
    ekv.rope_append_reference_paged(q, k, v, m.cs, m.kb, m.vb, m.table, ints([10, 10]), ints([0, 40, 50]))
    ekv.rope_append_paged(q, k, v, m.cs, m.kc, m.vc, m.table, ints([10, 10]), ints([-5, 40, 20]))
    torch.cuda.synchronize()
    kernels.check_status()
    assert same_bits(before[0, m.table[1].long()[0] * 16:][:10], m.kb[0, m.table[1].long()[0] * 16:][:10])


@pytest.mark.gpu
def test_offsets_that_do_not_ascend_stay_in_their_sequences_pages():
    """With offsets 0, 0, 736, 1000, 0 the page slots of sequence 2 begin at 736 / 16 +
    4 = 50, but two ends (2 and 8) lie before slots 8 to 49 as well: taken for its
    pages they would be pages -42 to -1, the last 42 of sequence 1's table row."""
    new, Hkv = [0, 736, 264, 0], 2
    q, k, v = tokens(1000, 4, Hkv, seed=97)
    m = Model(4, Hkv, 64, seed=15)
    cu = ints([0, 0, 736, 1000, 0])
    for c in (m.kc, m.vc):
        c.sm.fill_(7), c.code.fill_(7), c.rowmask.fill_(7), c.base.fill_(7)
    m.kb.fill_(7.0), m.vb.fill_(7.0)
    ekv.rope_append_paged(q, k, v, m.cs, m.kc, m.vc, m.table, ints(new), cu)
    ekv.rope_append_reference_paged(q, k, v, m.cs, m.kb, m.vb, m.table, ints(new), cu)
    kernels.check_status()
    theirs = torch.cat([m.table[b, :-(-n // 16)] for b, n in enumerate(new)]).long()
    other = torch.ones(m.pages, dtype=torch.bool, device="cuda")
    other[theirs] = False
    for c, bf in ((m.kc, m.kb), (m.vc, m.vb)):
        assert (c.rowmask[0, other] == 7).all() and (c.base[0, other] == 7).all()
        assert (c.sm.view(m.pages, -1)[other] == 7).all() and (c.code.view(m.pages, -1)[other] == 7).all()
        assert (bf.view(m.pages, -1)[other] == 7).all()


@pytest.mark.gpu
def test_full_raw_pool_drops_rows_past_its_capacity():
    """Slots past the capacity are not written: nothing beyond the pool changes, and
    the counter tells how many rows wanted one. A value far below its page's in
    one channel escapes when it is a value; the rotation of a key mixes it with
    the pair's other channel, so it need not."""
    Hkv = 2
    q, k, v = tokens(32, 4, Hkv, seed=95)
    k[::2, :, 3] = 1e-30
    m = Model(1, Hkv, 2, seed=5)
    c = m.kc.buffers()
    c["cap"], c["raw"] = 10, torch.full((10 + Hkv * 16, D), 3.0, dtype=torch.bfloat16, device="cuda")
    ekv.rope_append_paged(q, k, v, m.cs, c, m.vc, m.table, ints([32]), offsets([32]))
    want = ocodec.encode(to_bits(rotated(k, m.cs[:32]))[None])["raw"]
    assert int(c["cnt"].item()) == len(want) and (c["raw"][10:] == 3).all()
    assert np.array_equal(to_bits(c["raw"][:len(want)]), want[:10])
    v2 = m.vc.buffers()
    v2["cnt"].zero_()
    v2["cap"], v2["raw"] = 10, torch.full((10 + Hkv * 16, D), 3.0, dtype=torch.bfloat16, device="cuda")
    ekv.rope_append_paged(q, k, k, m.cs, m.kc, v2, m.table, ints([32]), offsets([32]))      # unrotated: every other row escapes
    want = ocodec.encode(to_bits(k)[None])["raw"]
    assert len(want) >= 32 and int(v2["cnt"].item()) == len(want) and (v2["raw"][10:] == 3).all()
    assert np.array_equal(to_bits(v2["raw"][:10]), want[:10])


@pytest.mark.gpu
def test_pool_growth_moves_open_pages():
    """ensure_headroom keeps every value, the open pages' among them, and the next
    steps go on."""
    m = Model(2, 2, 16, seed=9)
    for c in (m.kc, m.vc):
        c.pool = type(c.pool)(2, 2, D, 64, c.dev)
        c._bind()
    for i, new in enumerate(([20, 3], [1, 40], [30, 30])):
        moved = m.kc.ensure_headroom(sum(new)) | m.vc.ensure_headroom(sum(new))
        m.append(new, 4, seed=200 + 10 * i)
        m.check()
    assert moved in (True, False) and m.kc.pool.moves > 0


@pytest.mark.gpu
def test_prompt_then_steps_with_the_attention_that_reads_them():
    """The operators together: prompts in two chunks, each appended and attended over
    the pages; then single tokens, appended and read by attention_paged, from a
    captured graph. Compressed and bf16 pools give the same bits throughout, and
    each result is within the attention's bound of the formula."""
    from test_prefill_gpu import reference
    Hq, Hkv, B, pages = 8, 4, 3, 40
    m = Model(B, Hkv, pages, seed=12)
    lens = [0] * B
    for step, new in enumerate(([200, 37, 5], [100, 300, 17])):
        q, k, v = tokens(sum(new), Hq, Hkv, seed=300 + step)
        lens = [a + b for a, b in zip(lens, new)]
        sl, cu = ints(lens), offsets(new)
        q1 = ekv.rope_append_paged(q, k, v, m.cs, m.kc, m.vc, m.table, sl, cu)
        q2 = ekv.rope_append_reference_paged(q, k, v, m.cs, m.kb, m.vb, m.table, sl, cu)
        o1 = ekv.attention_prefill_paged(q1, m.kc, m.vc, m.table, sl, cu)
        o2 = ekv.attention_prefill_reference_paged(q2, m.kb, m.vb, m.table, sl, cu)
        assert same_bits(o1, o2)
        at = 0
        for b, n in enumerate(new):
            p = torch.arange(lens[b] - n, lens[b])
            m.k[b] = torch.cat([m.k[b], rotated(k[at:at + n], m.cs.cpu()[p])])
            m.v[b] = torch.cat([m.v[b], v[at:at + n].cpu()])
            at += n
        o, tol = reference(q1, torch.cat(m.k), torch.cat(m.v), new, lens)
        assert ((o1.double().cpu() - o).abs() <= tol).all()
    q, k, v = tokens(B, Hq, Hkv, seed=400)
    sl = ints(lens)
    outs = [torch.zeros(B, Hq, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]

    def step():
        sl.add_(1)
        q1 = ekv.rope_append_paged(q, k, v, m.cs, m.kc, m.vc, m.table, sl)
        q2 = ekv.rope_append_reference_paged(q, k, v, m.cs, m.kb, m.vb, m.table, sl)
        kernels.attention_paged(q1, m.kc, m.vc, m.table, sl, out=outs[0])
        kernels.attention_reference_paged(q2, m.kb, m.vb, m.table, sl, out=outs[1])

    graph = None
    for i in range(40):                                 # over page boundaries
        q0, k0, v0 = tokens(B, Hq, Hkv, seed=500 + 3 * i)
        q.copy_(q0), k.copy_(k0), v.copy_(v0)
        if i == 0:
            step()
        else:
            if graph is None:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    step()
            graph.replay()
        assert same_bits(*outs)
        for b in range(B):
            m.k[b] = torch.cat([m.k[b], rotated(k[b:b + 1], m.cs.cpu()[lens[b]:lens[b] + 1])])
            m.v[b] = torch.cat([m.v[b], v[b:b + 1].cpu()])
            lens[b] += 1
        if i % 13 == 0:
            qr = torch.cat([rotated(q[b:b + 1], m.cs.cpu()[lens[b] - 1:lens[b]]) for b in range(B)])
            o, tol = reference(qr, torch.cat(m.k), torch.cat(m.v), [1] * B, lens)
            assert ((outs[0].double().cpu() - o).abs() <= tol).all()
    assert sl.tolist() == lens
    kernels.check_status()


def test_rope_table_angles_in_64_bits():
    inv = THETA ** (-torch.arange(64, dtype=torch.float64) / 64)
    t = ekv.rope_table(inv.float(), 100000, scale=1.5)
    want = 99999.0 * inv.float().double()
    assert t.shape == (100000, D) and t.dtype == torch.float32
    assert torch.equal(t[99999], (1.5 * torch.cat([want.cos(), want.sin()])).float())
    with pytest.raises(ValueError):
        ekv.rope_table(inv[:32], 10)


def test_refusals():
    """Arguments that do not fit are refused on the host (CPU tensors: nothing runs)."""
    q = torch.zeros(4, 8, D, dtype=torch.bfloat16)
    k = torch.zeros(4, 2, D, dtype=torch.bfloat16)
    pool = torch.zeros(1, 64, 2, D, dtype=torch.bfloat16)
    i4 = torch.zeros(4, dtype=torch.int32)
    cs = table_of(64, "cpu")
    table = torch.zeros(4, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ekv.rope_append_reference_paged(q, k, k, cs, pool, pool, table, i4)
    with pytest.raises(ValueError, match="pools"):
        ekv.rope_append_reference_paged(q, k, k, cs, pool, pool[:, :32], table, i4)
    with pytest.raises(ValueError, match="multiple of 16"):
        ekv.rope_append_reference_paged(q, k, k, cs, pool[:, :20].contiguous(), pool[:, :20].contiguous(), table, i4)
    with pytest.raises(ValueError):
        ekv.PagedCompressedKV(0, 2, D, 1, device="cpu")


def test_entry_points_refuse_before_any_launch():
    """Argument errors of the C entries come back as codes (addresses never touched)."""
    import ctypes
    from exactkv_b200._lib import APPEND, PREFILL, CView, lib
    at = 1 << 40
    names = ("q k v q_out q_st q_sh k_st k_sh v_st v_sh o_st o_sh cos_sin q_norm k_norm cu_seqlens seq_lens block_table "
             "slots N B Hq Hkv rope_rows max_pages pool_pages eps").split()
    fits = dict(zip(names, (at, at, at, at, 1024, 128, 256, 128, 256, 128, 1024, 128, at, 0, 0, 0, at, at, 0, 4, 4, 8, 2,
                            64, 4, 16, 1e-6)))

    def app(**kw):
        return APPEND.pack(*{**fits, **{n: v or 0 for n, v in kw.items()}}.values())

    bf = lambda a, k=at: lib.exk_rope_append_bf16(a, k, 2 * at, None, 0, None)  # noqa: E731
    assert lib.exk_rope_append_bf16(None, at, at, None, 0, None) == -1
    for kw in (dict(q=None), dict(B=0), dict(Hq=7), dict(N=5), dict(q_norm=at), dict(max_pages=0), dict(pool_pages=0),
               dict(seq_lens=None), dict(rope_rows=0), dict(N=-1)):
        assert bf(app(**kw)) == -1, kw
    assert bf(app(q_st=1028)) == -2 and bf(app(k=at + 8)) == -2 and bf(app(), at + 2) == -2 and bf(app(), None) == -1 and bf(app(), 2 * at) == -1
    n = lib.exk_rope_append_scratch(4, 4, 2, 0)
    cv, other = (CView(x, x, x, x, x, x, 1000 + 4 * 2 * 16) for x in (at, 2 * at))
    short = CView(at, at, at, at, at, at, 1000 + 3 * 2 * 16)

    def coded(a=None, k=cv, cap=1000, scratch=at, bytes_=n, cnt=at):
        return lib.exk_rope_append_compressed(a or app(), ctypes.byref(k), cap, cnt, ctypes.byref(other), 1000, 2 * at,
                                              scratch, bytes_, None, 0, None)

    assert coded(bytes_=n - 1) == -1 and coded(k=short) == -1 and coded(cap=-1) == -1 and coded(scratch=None) == -1
    assert coded(scratch=at + 4) == -2 and coded(a=app(Hq=7)) == -1
    assert coded(k=other) == -1 and coded(cnt=2 * at) == -1      # one pool, or one counter, for keys and values

    pnames = "q out q_st q_sh o_st o_sh cu_q po pm pl N B Hq Hkv ns qk_scale".split()
    pfits = dict(zip(pnames, (at, at, 1024, 128, 1024, 128, at, 0, 0, 0, 4, 1, 8, 2, 1, 0.1)))

    def pre(**kw):
        p = PREFILL.pack(*{**pfits, **{n: v or 0 for n, v in kw.items()}}.values())
        return lib.exk_attention_prefill(p, at, 256, 128, at, 256, 128, 4, at, None, 0, None)

    for kw in (dict(q=None), dict(B=0), dict(Hq=7), dict(ns=0), dict(ns=2), dict(q_st=0), dict(cu_q=None),
               dict(ns=65), dict(B=65536), dict(N=65535 * 64)):
        assert pre(**kw) == -1, kw
    assert pre(Hq=34, Hkv=2) == -5 and pre(q_sh=132) == -2 and pre(out=at + 8) == -2
    assert lib.exk_prefill_splits(2, 1, 8, 2, 9000, 148) > 1 and lib.exk_prefill_splits(9000, 1, 8, 2, 9000, 148) == 1
    assert lib.exk_prefill_splits(2, 1, 8, 3, 9000, 148) == -1 and lib.exk_prefill_splits(2, 1, 34, 2, 9000, 148) == -5
