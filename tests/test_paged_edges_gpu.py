"""Paged appends and prompt attention where a call meets the pools' and the
batch's limits: raw pools that run out and are cleaned up, sequences that are cut
back, bad table entries beside good ones, offsets that are no batch's, values that
are not finite under weights that vanish, and which keys a row sees, key by key.
"""
import pytest
import torch

import exactkv_b200 as ekv
from exactkv_b200 import kernels
from gpu_util import same_bits
from test_prefill_gpu import inputs, reference
from test_rope_append_gpu import Model, ints, offsets, rotated, tokens

D = 128


def escaping(k, v, every=1, phase=0):
    """Every `every`-th row with one channel (of keys: one rotated pair) far below the other
    rows': it does not fit the code and is kept raw. Two channels by turns, so
    that neither is small in a whole page."""
    for i, c in enumerate((3, 5)):
        at = (i + phase) % 2 * every
        k[at::2 * every, :, c] = k[at::2 * every, :, c + 64] = 1e-30
        v[at::2 * every, :, c] = 1e-30


def append_both(m, q, k, v, lens, new, slots=None, **kw):
    sl, cu = ints(lens), offsets(new)
    a = ekv.rope_append_paged(q, k, v, m.cs, m.kc, m.vc, m.table, sl, cu, slots=slots, **kw)
    b = ekv.rope_append_reference_paged(q, k, v, m.cs, m.kb, m.vb, m.table, sl, cu, **kw)
    assert same_bits(a, b)
    return a


def rows_of(m, b, n, first=0):
    pos = torch.arange(first, n, device="cuda")
    return m.table[b].long()[pos // 16] * 16 + pos % 16


def decoded(c):
    return kernels.decode_to_bf16(c.buffers(), c.TS).flatten(0, 1)


def check_same_pools(m, lens):
    for c, bf in ((m.kc, m.kb), (m.vc, m.vb)):
        got = decoded(c)
        for b, n in enumerate(lens):
            r = rows_of(m, b, n)
            assert same_bits(got[r], bf[0][r]), b


# ----------------------------------------------------------------------------- raw pools

@pytest.mark.gpu
def test_pages_without_room_in_the_raw_pool_are_refused_by_readers():
    """40 slots for 256 raw rows, beside another sequence's open page in the rows behind
    them: the pages that have no room read as such (zeros in the raw rows, reported),
    never as the other sequence's rows; the pages that have room, and the other
    sequence, are right and report nothing. The host's checks then refuse to go on."""
    Hq, Hkv, new = 8, 4, [3, 64]
    m = Model(2, Hkv, 4, seed=31)
    q, k, v = tokens(67, Hq, Hkv, seed=700)
    escaping(k, v)
    m.vc.pool = type(m.vc.pool)(2, Hkv, D, 40, m.vc.dev)
    m.vc._bind()
    qr = append_both(m, q, k, v, new, new)
    kernels.check_status()
    assert int(m.vc.cnt.item()) == 4 * 16 * Hkv
    ro = m.vc.rowoff[0][m.table[1].long()].cpu()
    assert ro[0, :2].tolist() == [0, 16] and (ro[0, 2:] < 0).all() and (ro[1:] < 0).all()
    got = decoded(m.vc)
    with pytest.raises(RuntimeError, match="raw pool"):
        kernels.check_status()
    first, rest = rows_of(m, 1, 16), rows_of(m, 1, 64, 16)
    assert same_bits(got[first][:, :2], m.vb[0][first][:, :2])
    assert (got[first][:, 2:] == 0).all() and (got[rest] == 0).all()
    sl, cu = ints(new), offsets(new)
    ekv.attention_prefill_paged(qr, m.kc, m.vc, m.table, sl, cu)
    with pytest.raises(RuntimeError, match="raw pool"):
        kernels.check_status()
    last = qr[[2, 66]].contiguous()
    kernels.attention_paged(last, m.kc, m.vc, m.table, sl)
    with pytest.raises(RuntimeError, match="raw pool"):
        kernels.check_status()
    only = offsets([3, 0])
    a = ekv.attention_prefill_paged(qr[:3], m.kc, m.vc, m.table, sl, only)
    assert same_bits(a, ekv.attention_prefill_reference_paged(qr[:3], m.kb, m.vb, m.table, sl, only))
    kernels.check_status()
    with pytest.raises(RuntimeError, match="raw rows"):
        m.vc.ensure_headroom(1)


# ----------------------------------------------------------------------------- what sequences hold

CUTS = [  # (tokens held, new tokens) of two sequences, call by call: fewer held than the call before left is a cut
    [(0, 45), (0, 20)],
    [(45, 5), (20, 14)],       # drafts that complete a page each and open the next
    [(46, 1), (25, 3)],        # cut back into the completed pages, which stay open
    [(47, 1), (28, 4)],        # ... and fill again
    [(48, 20), (32, 40)],
    [(40, 30), (33, 1)],       # into a page that this call completes before it opens another; by two pages
    [(5, 3), (34, 60)],
    [(8, 8), (94, 0)],
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["paged", "contiguous", "slots"])
@pytest.mark.parametrize("every", [1, 3, 1000])
def test_sequences_cut_back_into_completed_pages(kind, every):
    """Rejected drafts: the lengths end inside a page that was completed and coded. Both pools hold the
    same rows after every cut and every call, and are attended with the same bits; also
    with a CompressedKV as the pool, and with other tail slots."""
    Hq, Hkv = 8, 4
    m = Model(2, Hkv, 8, spare=0, seed=33, tails=5)
    slots = None
    if kind == "contiguous":
        m.kc, m.vc = (ekv.CompressedKV(2, 128, Hkv, D, reserve=2.0) for _ in range(2))
    else:
        slots = ints([3, 1]) if kind == "slots" else None
        for c in (m.kc, m.vc):
            c.ensure_headroom(2000)
    for i, call in enumerate(CUTS):
        lens, new = [h + n for h, n in call], [n for _, n in call]
        q, k, v = tokens(sum(new), Hq, Hkv, seed=710 + 3 * i)
        escaping(k, v, every)
        held = [h for h, _ in call]
        if i and held != left:
            ekv.cut_back_paged(m.kc, m.vc, m.table, ints(held), slots)
            check_same_pools(m, held)
            before = [t.clone() for c in (m.kc, m.vc) for t in (c.raw, c.rowmask, c.rowoff)]
            ekv.cut_back_paged(m.kc, m.vc, m.table, ints(held), slots)      # nothing is left to do
            assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in
                       zip(before, [t for c in (m.kc, m.vc) for t in (c.raw, c.rowmask, c.rowoff)]))
        left = lens
        qr = append_both(m, q, k, v, lens, new, slots)
        check_same_pools(m, lens)
        sl, cu = ints(lens), offsets(new)
        a = ekv.attention_prefill_paged(qr, m.kc, m.vc, m.table, sl, cu)
        assert same_bits(a, ekv.attention_prefill_reference_paged(qr, m.kb, m.vb, m.table, sl, cu))
        q1 = torch.randn(2, Hq, D, device="cuda").to(torch.bfloat16)
        a = kernels.attention_paged(q1, m.kc, m.vc, m.table, sl)
        assert same_bits(a, kernels.attention_reference_paged(q1, m.kb, m.vb, m.table, sl))
        kernels.check_status()
    assert int(m.vc.cnt.item()) > (0 if every == 1000 else 100)


@pytest.mark.gpu
def test_cut_back_in_a_captured_step_and_out_of_range():
    """Captured: it follows the lengths on the device. Lengths, pages and slots out of
    range are reported, and nothing of their sequences changes."""
    Hq, Hkv, B = 4, 2, 3
    m = Model(B, Hkv, 3, seed=34)
    q, k, v = tokens(3 * 40, Hq, Hkv, seed=735)
    escaping(k, v, 2)
    append_both(m, q, k, v, [40] * 3, [40] * 3)
    sl = ints([40] * 3)
    ekv.cut_back_paged(m.kc, m.vc, m.table, sl)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ekv.cut_back_paged(m.kc, m.vc, m.table, sl)
    bad = m.table.clone()
    bad[2, 1] = -4
    for lens, table, slots, match in (([49, 0, -7], m.table, None, "length"), ([40, 40, 20], bad, None, "outside the pool"),
                                      ([20, 40, 40], m.table, [3, 1, 2], "tail slot")):
        before = [t.clone() for c in (m.kc, m.vc) for t in (c.raw, c.rowmask, c.rowoff)]
        ekv.cut_back_paged(m.kc, m.vc, table, ints(lens), None if slots is None else ints(slots))
        with pytest.raises(RuntimeError, match=match):
            kernels.check_status()
        assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in
                   zip(before, [t for c in (m.kc, m.vc) for t in (c.raw, c.rowmask, c.rowoff)]))
    lens = [17, 32, 5]
    sl.copy_(ints(lens))
    graph.replay()
    kernels.check_status()
    check_same_pools(m, lens)
    q, k, v = tokens(3 * 30, Hq, Hkv, seed=738)
    lens = [n + 30 for n in lens[:1]] + [lens[1], lens[2] + 4]
    append_both(m, q[:34], k[:34], v[:34], lens, [30, 0, 4])
    check_same_pools(m, lens)
    kernels.check_status()


def test_cut_back_refusals():
    """On the host, before any launch (addresses never touched)."""
    import ctypes
    from exactkv_b200._lib import CView, lib
    at = 1 << 40
    kc, vc, short = (CView(x, x, x, x, x, x, n) for x, n in ((at, 1000 + 4 * 32), (2 * at, 1000 + 4 * 32), (at, 1000 + 3 * 32)))
    fits = dict(table=at, B=4, max_pages=4, pages=16, H=2, lens=at, slots=None, k=kc, k_cap=1000, v=vc, v_cap=1000)

    def call(**kw):
        a = {**fits, **kw}
        for n in ("k", "v"):
            a[n] = None if a[n] is None else ctypes.byref(a[n])
        return lib.exk_reopen_pages(*a.values(), None, 0, None)

    for kw in (dict(table=None), dict(B=0), dict(max_pages=0), dict(pages=0), dict(H=0), dict(lens=None), dict(k=None),
               dict(v=kc), dict(k=short), dict(k_cap=-1), dict(v_cap=2000), dict(pages=1 << 30, H=4)):
        assert call(**kw) == -1, kw
    assert call(k=CView(at + 4, at, at, at, at, at, 1000 + 4 * 32)) == -2
    pool = ekv.PagedCompressedKV(4, 2, D, 2, device="cpu")
    for args in ((pool, pool, torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)),
                 (pool, ekv.PagedCompressedKV(5, 2, D, 2, device="cpu"), torch.zeros(2, 4, dtype=torch.int32),
                  torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError):
            ekv.cut_back_paged(*args)


@pytest.mark.gpu
def test_open_page_is_written_beside_a_bad_entry():
    """A call that would complete a page whose entry is bad and opens another: the good
    entries' pages hold what the bf16 pool holds."""
    Hq, Hkv = 4, 2
    m = Model(1, Hkv, 4, seed=35)
    q, k, v = tokens(20, Hq, Hkv, seed=740)
    append_both(m, q, k, v, [20], [20])
    good = m.table.clone()
    m.table[0, 1] = m.pages
    q, k, v = tokens(30, Hq, Hkv, seed=743)
    append_both(m, q, k, v, [50], [30])
    with pytest.raises(RuntimeError, match="outside the pool"):
        kernels.check_status()
    m.table = good
    for c, bf in ((m.kc, m.kb), (m.vc, m.vb)):
        got = decoded(c)
        for lo, hi in ((0, 16), (32, 48), (48, 50)):
            r = rows_of(m, 0, hi, lo)
            assert same_bits(got[r], bf[0][r]), lo
    kernels.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[16 * 40] * 32, [13] * 1300, [31] * 520])
def test_normed_keys_have_the_same_bits_in_both_pools(lens):
    """Over 1e5 normed heads a pool, in encoded pages, among them raw rows, and in open
    pages: one order of the sum of squares for every path."""
    Hkv, B = 8, len(lens)
    n = sum(lens)
    m = Model(B, Hkv, -(-max(lens) // 16), seed=37)
    g = torch.Generator(device="cuda").manual_seed(38)
    wq, wk = (torch.randn(D, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    q, k, v = tokens(n, Hkv, Hkv, seed=750)
    escaping(k, v, 5)
    append_both(m, q, k, v, lens, lens, q_norm=wq, k_norm=wk)
    kernels.check_status()
    assert n * Hkv >= 100000 and (max(lens) < 16 or int(m.kc.cnt.item()) > 1000)
    at = torch.cat([rows_of(m, b, m_) for b, m_ in enumerate(lens)])
    got = decoded(m.kc)
    assert same_bits(got[at], m.kb[0][at])
    assert same_bits(decoded(m.vc)[at], v)


@pytest.mark.gpu
def test_normed_keys_and_queries_one_token_at_a_time():
    """The same bits as the whole prompt gives, and within the norm's bound of the formula."""
    Hq, Hkv, B, n = 8, 8, 400, 33
    m, whole = (Model(B, Hkv, 3, seed=39) for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(40)
    w = dict(zip(("q_norm", "k_norm"), (torch.randn(D, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))))
    q, k, v = tokens(B * n, Hq, Hkv, seed=760)
    escaping(k, v, 7)
    qw = append_both(whole, q, k, v, [n] * B, [n] * B, **w).view(B, n, Hq, D)
    parts = [t.view(B, n, -1, D) for t in (q, k, v)]
    for i in range(n):
        one = [t[:, i].contiguous() for t in parts]
        sl = ints([i + 1] * B)
        a = ekv.rope_append_paged(*one, m.cs, m.kc, m.vc, m.table, sl, **w)
        b = ekv.rope_append_reference_paged(*one, m.cs, m.kb, m.vb, m.table, sl, **w)
        assert same_bits(a, b) and same_bits(a, qw[:, i].contiguous())
    kernels.check_status()
    at = torch.cat([rows_of(m, b, n) for b in range(B)])
    assert same_bits(m.kb, whole.kb)
    for c in (m.kc, whole.kc):
        assert same_bits(decoded(c)[at], m.kb[0][at])
    some = torch.arange(0, B * n, 97)
    y, tol = rotated(k[some.cuda()], m.cs.cpu()[some % n], w["k_norm"])
    assert ((m.kb[0][at][some.cuda()].double().cpu() - y).abs() <= tol).all()


def test_norm_weights_off_their_alignment_are_refused():
    """The kernels read them 8 bytes at a time: a view into a flat buffer of weights may
    begin anywhere. Refused by the C entries before any launch (addresses never touched)."""
    import ctypes
    from exactkv_b200._lib import APPEND, CView, lib
    at = 1 << 40
    fits = [at, at, at, at, 1024, 128, 256, 128, 256, 128, 1024, 128, at, at, at, 0, at, at, 0, 4, 4, 8, 2, 64, 4, 16, 1e-6]
    pools = [ctypes.byref(CView(x, x, x, x, x, x, 1000 + 4 * 32)) for x in (at, 2 * at)]
    n = lib.exk_rope_append_scratch(4, 4, 2, 0)
    for which in (13, 14):
        for off in (2, 4, 6):
            a = APPEND.pack(*[x + off if i == which else x for i, x in enumerate(fits)])
            assert lib.exk_rope_append_bf16(a, at, 2 * at, None, 0, None) == -2
            assert lib.exk_rope_append_compressed(a, pools[0], 1000, at, pools[1], 1000, 2 * at, at, n, None, 0, None) == -2


@pytest.mark.gpu
def test_norm_weights_may_be_aligned_views_and_no_others():
    Hkv = 2
    m = Model(1, Hkv, 2, seed=41)
    q, k, v = tokens(20, 4, Hkv, seed=765)
    flat = torch.randn(3 * D, device="cuda").to(torch.bfloat16)
    sl, cu = ints([20]), offsets([20])
    for off, fits in ((8, True), (4, True), (1, False), (6, False)):
        w = flat[off:off + D]
        for call, pools in ((ekv.rope_append_paged, (m.kc, m.vc)), (ekv.rope_append_reference_paged, (m.kb, m.vb))):
            if not fits:
                with pytest.raises(ValueError, match="8-byte"):
                    call(q, k, v, m.cs, *pools, m.table, sl, cu, q_norm=w, k_norm=w)
                continue
            got = call(q, k, v, m.cs, *pools, m.table, sl, cu, q_norm=w, k_norm=w)
            y, tol = rotated(q, m.cs[:20], w)
            assert ((got.double().cpu() - y).abs() <= tol).all()
    kernels.check_status()


# ----------------------------------------------------------------------------- offsets

@pytest.mark.gpu
@pytest.mark.parametrize("klen,seqs", [(40, 3), (3000, 3), (3000, 40)])
def test_offsets_that_are_no_batchs_are_reported_and_leave_rows_alone(klen, seqs):
    """Rows of a sequence whose offsets leave the batch or descend are not written, with
    and without splits (where nothing wrote the partials that would be merged), and
    the call is reported; so are such offsets of the keys."""
    Hq, Hkv, N = 8, 2, 20
    lens = [12] + [0] * (seqs - 3) + [4, 4]
    bad = offsets(lens)
    bad[-2] = 30                                     # 0, 12, .., 12, 30, 20: past the queries, then descending
    q, k, v = inputs(N, klen * seqs, Hq, Hkv, seed=42)
    ck = offsets([klen] * seqs)
    plan = kernels.lib.exk_prefill_splits(N, seqs, Hq, Hkv, klen, kernels.num_sms())
    assert (plan > 1) == (klen > 1000)
    good = offsets(lens)
    want = ekv.attention_prefill(q, k, v, good, ck)
    kernels.check_status()
    junk = torch.full((N * Hq * plan * (D + 2),), float("nan"), device="cuda")
    del junk                                         # (what the call's workspace may find)
    hold = torch.full_like(q, 5.0)
    ekv.attention_prefill(q, k, v, bad, ck, out=hold)
    assert (hold[12:] == 5).all()
    assert same_bits(hold[:12], want[:12]) or (hold[:12] == 5).all()
    with pytest.raises(RuntimeError, match="offsets"):
        kernels.check_status()
    for at, x in ((0, -1), (1, 2 * klen + 1), (seqs, klen * seqs + 1)):
        wrong = ck.clone()
        wrong[at] = x
        ekv.attention_prefill(q, k, v, good, wrong)
        with pytest.raises(RuntimeError, match="offsets"):
            kernels.check_status()


# ----------------------------------------------------------------------------- values

@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("lens,klens,cold,hot", [
    ([4], [5000], 10, 4990), ([4], [5000], 4990, 10), ([4], [5000], 2500, 2501), ([300], [300], 10, 200),
    ([300], [300], 200, 10), ([300], [600], 590, 3)])
def test_value_that_is_not_finite_under_a_weight_that_vanishes(lens, klens, cold, hot, bad):
    """Scores 350 apart: the key's weight is exp(-350) in the formula and underflows in 32
    bits. The rows that see it are not finite in its channel, whatever the tile, the mask
    and the splits; every other value keeps its bits."""
    Hq, Hkv, n, L = 8, 2, lens[0], klens[0]
    q, k, v = inputs(n, L, Hq, Hkv, seed=44)
    q.zero_(), k.zero_()
    q[..., 0] = 8
    k[hot, :, 0] = 500
    cu, ck = offsets(lens), offsets(klens)
    clean = ekv.attention_prefill(q, k, v, cu, ck)
    o, tol = reference(q, k, v, lens, klens)
    assert ((clean.double().cpu() - o).abs() <= tol).all()
    v[cold, 1, 77] = bad
    out = ekv.attention_prefill(q, k, v, cu, ck)
    hit = torch.zeros(n, Hq, D, dtype=torch.bool, device="cuda")
    hit[max(0, cold - (L - n)):, 4:, 77] = True
    assert torch.equal(~torch.isfinite(out.float()), hit)
    assert same_bits(torch.where(hit, 0, out), torch.where(hit, 0, clean))


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_channels_beside_a_value_that_is_not_finite_keep_their_bits(bad):
    Hq, Hkv = 8, 2
    for lens, klens, at in (([300], [300], 150), ([20, 30], [20, 30], 12), ([4], [5000], 4998), ([4], [5000], 700)):
        q, k, v = inputs(sum(lens), sum(klens), Hq, Hkv, seed=46)
        cu, ck = offsets(lens), offsets(klens)
        clean = ekv.attention_prefill(q, k, v, cu, ck)
        v[at, 1, 77] = bad
        out = ekv.attention_prefill(q, k, v, cu, ck)
        out[:, 4:, 77] = clean[:, 4:, 77]
        assert same_bits(out, clean)


SEEN = [([300], [300]), ([300], [1000]), ([1, 40, 129], [1, 333, 2049]), ([3], [9000]), ([50], [4097]), ([5, 2, 9], [6000, 4095, 1000])]


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (7, 1), (28, 4)])
@pytest.mark.parametrize("case", range(len(SEEN)))
def test_each_row_sees_each_key_once(case, Hq, Hkv):
    """Scores of zero and values that are 1 in one channel of one key: a row's output is
    1 / (its keys) in the channels of the keys that it sees, once each, and 0 elsewhere.
    128 keys at a time: the ends of tiles, pages and splits, the first and the last, and
    others. With p = 1 and whole sums the only roundings are the quotient's: 2^-8 for
    bf16, 2^-20 for the 32 bits before it."""
    lens, klens = SEEN[case]
    g = torch.Generator().manual_seed(case)
    N, Nk = sum(lens), sum(klens)
    m = Model(len(lens), Hkv, -(-max(klens) // 16), seed=50 + case)
    q = torch.zeros(N, Hq, D, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(Nk, Hkv, D, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    chosen, at = [], 0
    for n, L in zip(lens, klens):
        edge = [0, 1, 15, 16, 17, 127, 128, 129, 255, 256, L - 1, L - 2, L - n, L - n - 1, L - n + 1, L - 129, L - 128, L - 17, L - 16]
        edge += [t * 128 + d for t in range(2, L // 128, max(1, L // 128 // 16)) for d in (-1, 0)]
        keys = [j for j in dict.fromkeys(edge) if 0 <= j < L][:D]
        keys += torch.randint(0, L, (D - len(keys),), generator=g).tolist()
        chosen.append(keys)
        v[at + torch.tensor(keys), :, torch.arange(D)] = 1
        at += L
    want, at = torch.zeros(N, D, dtype=torch.float64), 0
    for b, (n, L) in enumerate(zip(lens, klens)):
        last = torch.arange(n) + L - n
        want[at:at + n] = (torch.tensor(chosen[b])[None] <= last[:, None]).double() / (last + 1)[:, None]
        at += n
    cu, ck, sl = offsets(lens), offsets(klens), ints(klens)
    append_both(m, k, k, v, klens, klens)
    outs = [ekv.attention_prefill(q, k, v, cu, ck), ekv.attention_prefill_paged(q, m.kc, m.vc, m.table, sl, cu),
            ekv.attention_prefill_reference_paged(q, m.kb, m.vb, m.table, sl, cu)]
    for out in outs:
        err = (out.double().cpu() - want[:, None]).abs()
        assert (err <= (2.0 ** -8 + 2.0 ** -20) * want[:, None]).all()
    kernels.check_status()


# ----------------------------------------------------------------------------- growing and cleaning up

@pytest.mark.gpu
def test_check_overflow_covers_paged_pools():
    """One call for all layers' pools, contiguous ones among them: those with less than a
    worst-case page for every sequence grow, and the next 16 steps fit."""
    Hq, Hkv, B = 4, 2, 3
    m = Model(B, Hkv, 8, seed=60)
    for c in (m.kc, m.vc):
        c.pool = type(c.pool)(B, Hkv, D, 64, c.dev)
        c._bind()
    flat = ekv.CompressedKV(B, 64, Hkv, D)
    new = [5, 14, 16]
    q, k, v = tokens(sum(new), Hq, Hkv, seed=770)
    escaping(k, v)
    grew = ekv.check_overflow([m.kc, flat, m.vc])
    assert grew == 2 and m.kc.cap >= 16 * B * Hkv and m.kc.pool.moves == 1
    append_both(m, q, k, v, new, new)
    lens = new
    for step in range(40):
        if step % 16 == 0:
            ekv.check_overflow([m.kc, m.vc])
        q, k, v = tokens(B, Hq, Hkv, seed=780 + 3 * step)
        escaping(k, v, phase=step)
        lens = [n + 1 for n in lens]
        append_both(m, q, k, v, lens, [1] * B)
        assert int(m.vc.cnt.item()) <= m.vc.cap
    assert int(m.vc.cnt.item()) > 100 and m.vc.pool.moves > 1
    assert ekv.check_overflow([]) == 0
    check_same_pools(m, lens)
    kernels.check_status()


@pytest.mark.gpu
def test_growth_moves_open_pages_and_keeps_every_row():
    Hq, Hkv, lens = 4, 2, [0, 0]
    m = Model(2, Hkv, 16, seed=62)
    for c in (m.kc, m.vc):
        c.pool = type(c.pool)(2, Hkv, D, 64, c.dev)
        c._bind()
    for i, new in enumerate(([20, 3], [1, 40], [60, 30])):
        moved = [c.ensure_headroom(sum(new)) for c in (m.kc, m.vc)]
        assert moved == [True, True] or i == 1
        q, k, v = tokens(sum(new), Hq, Hkv, seed=900 + 3 * i)
        escaping(k, v)
        lens = [a + b for a, b in zip(lens, new)]
        append_both(m, q, k, v, lens, new)
        check_same_pools(m, lens)
    assert m.kc.pool.moves >= 2
    kernels.check_status()


@pytest.mark.gpu
def test_raw_rows_of_freed_pages_are_given_back():
    """Sequences come and go on a pool's pages; compact() keeps the raw rows of the pages
    in use, so the raw pool stays as it is. Open pages and pages shared by two tables
    are kept, and the storage does not move."""
    Hq, Hkv = 4, 2
    m = Model(3, Hkv, 4, seed=64)
    lens = [0, 0, 0]
    for c in (m.kc, m.vc):
        c.ensure_headroom(400)
    at = [c.pool.rows.data_ptr() for c in (m.kc, m.vc)]
    for turn in range(12):
        gone = turn % 3                                  # this sequence ends; its pages and its slot go to another
        lens[gone] = 0
        new = [0, 0, 0]
        new[gone] = 21 + turn
        new[(gone + 1) % 3] = 1
        q, k, v = tokens(sum(new), Hq, Hkv, seed=920 + 3 * turn)
        escaping(k, v, 1 + turn % 2)
        live = torch.cat([torch.cat([m.table[b, :-(-n // 16)], ints([-1])]) for b, n in enumerate(lens)])
        live = torch.cat([live, live]).view(2, -1)       # as two tables that share every page
        for c in (m.kc, m.vc):
            used = int(c.cnt.item())
            kept = c.compact(live)
            assert kept == int(c.cnt.item()) <= used
        check_same_pools(m, lens)
        lens = [a + b for a, b in zip(lens, new)]
        append_both(m, q, k, v, lens, new)
        check_same_pools(m, lens)
        assert int(m.vc.cnt.item()) <= 3 * 64 * Hkv
    assert at == [c.pool.rows.data_ptr() for c in (m.kc, m.vc)]
    # a pool that ran out goes on without the pages that had no room
    live = m.table[0, :-(-lens[0] // 16)]
    m.vc.cnt.fill_(m.vc.cap + 1)
    with pytest.raises(RuntimeError, match="raw rows"):
        ekv.check_overflow([m.vc])
    assert m.vc.compact(live) <= 64 * Hkv and not m.vc.ensure_headroom(64)
    m.kc.compact(live)
    check_same_pools(m, lens[:1])
    for c in (m.kc, m.vc):
        assert c.compact(m.table[:0]) == 0
    kernels.check_status()


@pytest.mark.gpu
def test_compact_with_pages_set_aside():
    """A table may name pages that its sequence has not come to yet. What an earlier sequence
    left in them is not taken for rows in use once the pool was cleaned up without it: the
    count never grows, and the open pages behind the capacity are not written over."""
    Hq, Hkv = 4, 2
    m = Model(2, Hkv, 4, seed=66)
    for c in (m.kc, m.vc):
        c.pool = type(c.pool)(2, Hkv, D, 140, c.dev)
        c._bind()
    q, k, v = tokens(64 + 20, Hq, Hkv, seed=960)
    escaping(k, v)
    append_both(m, q[:64], k[:64], v[:64], [64, 0], [64, 0])
    lens = [0, 5]
    for c in (m.kc, m.vc):
        assert c.compact(m.table[1]) == 0                # sequence 0 has ended
    append_both(m, q[64:69], k[64:69], v[64:69], lens, [0, 5])
    check_same_pools(m, lens)
    for n in (15, 12, 17):                               # sequence 1 goes on; 0's pages are set aside for another
        q, k, v = tokens(n, Hq, Hkv, seed=970 + n)
        escaping(k, v)
        lens = [0, lens[1] + n]
        append_both(m, q, k, v, lens, [0, n])
        for c in (m.kc, m.vc):
            used = int(c.cnt.item())
            assert c.compact(m.table) <= used
        check_same_pools(m, lens)
    kernels.check_status()
