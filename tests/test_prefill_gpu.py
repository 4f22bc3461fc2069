"""Prompt attention (exk_attention_prefill, over pages, over compressed pages)
against the formula in 64 bits.

Every comparison allows, per output,
    (2^-8 + 2 d) sum_j p_j |v_j| + 2^-8 |o| + 2^-20 sum_j p_j |v_j|
: P is rounded to bf16 before the product (half a step, 2^-8 of each term), the
output once more (2^-8 |o|), sums are held in 32 bits (2^-20), and a score
carries an error of at most d = 130 * 2^-23 max_j sum_c |q_c k_jc| / sqrt(128)
(128 products added in fp32, in any order, each step truncated at worst),
which moves p_j and the normaliser by the factor exp(d) each.
"""
import numpy as np
import pytest
import torch

import exactkv_b200 as ekv
from exactkv_b200 import kernels, synthetic
from gpu_util import same_bits

D = 128


def offsets(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32)


def reference(q, k, v, lens, klens):
    """(o, tolerance) in float64 on the CPU; rows without keys are zero."""
    q, k, v = (t.double().cpu() for t in (q, k, v))
    Hq, Hkv = q.shape[1], k.shape[1]
    G = Hq // Hkv
    o, tol = torch.zeros_like(q), torch.zeros_like(q)
    a = b = 0
    for n, L in zip(lens, klens):
        if n and L:
            qs = q[a:a + n].view(n, Hkv, G, D)
            ks, vs = k[b:b + L], v[b:b + L]
            sees = torch.arange(L)[None] <= torch.arange(n)[:, None] + L - n
            s = torch.einsum("nhgd,lhd->nhgl", qs, ks) / D ** 0.5
            mag = (torch.einsum("nhgd,lhd->nhgl", qs.abs(), ks.abs()) / D ** 0.5)
            hide = ~sees[:, None, None]
            s = s.masked_fill(hide, -torch.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.where(hide, 0.0, (s - torch.where(top.isinf(), 0.0, top)).exp())
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            out = torch.einsum("nhgl,lhd->nhgd", p, vs)
            av = torch.einsum("nhgl,lhd->nhgd", p, vs.abs())
            d = 130 * 2.0 ** -23 * mag.masked_fill(hide, 0.0).amax(-1)[..., None]
            o[a:a + n] = out.reshape(n, Hq, D)
            tol[a:a + n] = ((2.0 ** -8 + 2.0 ** -20 + 2 * d) * av + 2.0 ** -8 * out.abs() + 1e-30).reshape(n, Hq, D)
        a, b = a + n, b + L
    return o, tol


def inputs(N, Nk, Hq, Hkv, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    mk = lambda n, h: (torch.randn(n, h, D, generator=g, device="cuda") * scale).to(torch.bfloat16)  # noqa: E731
    return mk(N, Hq), mk(Nk, Hkv), mk(Nk, Hkv)


def check(out, q, k, v, lens, klens):
    o, tol = reference(q, k, v, lens, klens)
    n = sum(lens)
    err = (out[:n].double().cpu() - o[:n]).abs()
    assert torch.isfinite(out[:n].float()).all()
    assert (err <= tol[:n]).all(), f"max err/tol {(err / tol[:n]).max():.3g}"


CASES = [
    # lens, key lens (None: the same)
    ([1], None),
    ([1, 2, 3], None),
    ([127, 128, 129], None),
    ([0, 5, 0, 300, 0], None),
    ([64, 1000, 17], None),
    ([700], None),
    ([3, 40], [130, 1000]),            # context before the queries
    ([1, 1], [1, 257]),
    ([40, 9, 6], [10, 0, 6]),          # queries that see no key, a sequence without keys
    ([2], [9000]),                     # few rows, many keys: split
    ([5, 1, 30], [4097, 2000, 3000]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (28, 4), (16, 1), (4, 4), (9, 3), (11, 1)])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_prefill_matches_formula(case, Hq, Hkv):
    lens, klens = CASES[case]
    same = klens is None
    klens = klens or lens
    q, k, v = inputs(sum(lens), sum(klens), Hq, Hkv, seed=case)
    out = ekv.attention_prefill(q, k, v, offsets(lens).cuda(), None if same else offsets(klens).cuda())
    check(out, q, k, v, lens, klens)
    kernels.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.05, 4.0])
def test_prefill_flat_and_peaked_scores(scale):
    """Scores near zero everywhere, and scores of +-200: the running maximum grows
    and rows are rescaled."""
    lens = [500, 260]
    q, k, v = inputs(760, 760, 8, 2, seed=7, scale=scale)
    k[:500] *= torch.linspace(2.0, 0.1, 500, device="cuda")[:, None, None].to(torch.bfloat16)   # grows towards key 0
    out = ekv.attention_prefill(q, k, v, offsets(lens).cuda())
    check(out, q, k, v, lens, lens)


@pytest.mark.gpu
def test_prefill_strided_views_and_rows_past_the_batch():
    """q, k, v as views of one fused projection, out a view too; rows past the last
    sequence keep what they held."""
    lens, Hq, Hkv = [100, 31], 8, 4
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(140, Hq + 2 * Hkv + 1, D, generator=g, device="cuda").to(torch.bfloat16)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:Hq + 2 * Hkv]
    hold = torch.full((140, 2 * Hq, D), 7.0, dtype=torch.bfloat16, device="cuda")
    out = ekv.attention_prefill(q, k, v, offsets(lens).cuda(), out=hold[:, ::2])
    check(out, q[:131], k[:131], v[:131], lens, lens)
    assert (hold[131:] == 7).all() and (hold[:, 1::2] == 7).all()
    dense = ekv.attention_prefill(q.contiguous(), k.contiguous(), v.contiguous(), offsets(lens).cuda())
    assert same_bits(out[:131], dense[:131])
    # head-major storage [heads, N, 128] seen as [N, heads, 128]
    qt, kt, vt = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    assert same_bits(ekv.attention_prefill(qt, kt, vt, offsets(lens).cuda())[:131], dense[:131])


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("lens,klens,at", [([300], [300], 150), ([20, 30], [20, 30], 12), ([4], [5000], 4998)])
def test_values_and_keys_that_are_not_finite_reach_only_the_rows_that_see_them(lens, klens, at, bad):
    """A non-finite value (or key) at key `at` of sequence 0: the rows before it,
    and the other sequences, keep their bits; rows that see the value get it in
    that channel and keep the others."""
    Hq, Hkv = 8, 2
    q, k, v = inputs(sum(lens), sum(klens), Hq, Hkv, seed=11)
    cu, ck = offsets(lens).cuda(), offsets(klens).cuda()
    clean = ekv.attention_prefill(q, k, v, cu, ck)
    first = max(0, at - (klens[0] - lens[0]))            # first row of sequence 0 that sees it
    sees = torch.zeros(sum(lens), dtype=torch.bool)
    sees[first:lens[0]] = True
    v2 = v.clone()
    v2[at, 1, 77] = bad
    out = ekv.attention_prefill(q, k, v2, cu, ck)
    assert same_bits(out[~sees], clean[~sees])
    hit = out[sees][:, 4:, 77].float()
    assert (hit.isnan() if bad != bad else hit == bad).all()
    keep = out[sees].clone()
    keep[:, 4:, 77] = clean[sees][:, 4:, 77]
    assert torch.isfinite(keep.float()).all() and ((keep - clean[sees]).float().abs() < 1).all()
    k2 = k.clone()
    k2[at, 0, 5] = bad
    out = ekv.attention_prefill(q, k2, v, cu, ck)
    assert same_bits(out[~sees], clean[~sees]) and same_bits(out[:, 4:], clean[:, 4:])
    # rows of a larger buffer behind the last key: whatever they hold, the same bits
    # (the plan of the splits goes by the buffer's size, so both calls have one)
    pad = lambda t, x: torch.cat([t, torch.full((200, Hkv, D), x, dtype=torch.bfloat16, device="cuda")])  # noqa: E731
    want = ekv.attention_prefill(q, pad(k, 1.0), pad(v, 1.0), cu, ck)
    assert same_bits(ekv.attention_prefill(q, pad(k, bad), pad(v, bad), cu, ck), want)
    check(want, q, k, v, lens, klens)


def _pools(lens, Hkv, seed, spare=5, max_extra=2):
    """The same sequences contiguous, in bf16 pools and in compressed pools."""
    k = synthetic.make_kv(1, sum(lens), Hkv, seed=seed, key=True, raw_frac=0.01)[0]
    v = synthetic.make_kv(1, sum(lens), Hkv, seed=seed + 1, key=False, raw_frac=0.01)[0]
    pages = [-(-n // 16) for n in lens]
    total = sum(pages) + spare
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).int()
    table = torch.full((len(lens), max(pages) + max_extra), -7, dtype=torch.int32)
    at = 0
    for b, m in enumerate(pages):
        table[b, :m] = perm[at:at + m]
        at += m
    table = table.cuda()
    kb, vb = (torch.full((1, total * 16, Hkv, D), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kc, vc = (ekv.PagedCompressedKV(total, Hkv, D, len(lens), reserve=1.0) for _ in range(2))
    ident = torch.cat([torch.ones(sum(lens), 64), torch.zeros(sum(lens), 64)], 1).cuda()     # no rotation
    q0 = torch.zeros(sum(lens), Hkv, D, dtype=torch.bfloat16, device="cuda")
    sl, cu = torch.tensor(lens, dtype=torch.int32, device="cuda"), offsets(lens).cuda()
    ekv.rope_append_reference_paged(q0, k, v, ident, kb, vb, table, sl, cu)
    ekv.rope_append_paged(q0, k, v, ident, kc, vc, table, sl, cu)
    kernels.check_status()
    return k, v, kb, vb, kc, vc, table, sl


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (28, 4), (5, 5)])
@pytest.mark.parametrize("lens,klens", [([1], [1]), ([3, 40, 1], [130, 1000, 16]), ([300, 17], [300, 2049]),
                                        ([6], [9000]), ([30, 5, 0], [10, 0, 33])])
def test_paged_equals_contiguous_bit_for_bit(lens, klens, Hq, Hkv):
    q, _, _ = inputs(sum(lens), 1, Hq, Hkv, seed=21)
    k, v, kb, vb, kc, vc, table, sl = _pools(klens, Hkv, seed=22)
    cu, ck = offsets(lens).cuda(), offsets(klens).cuda()
    most = max(klens)
    o_b = ekv.attention_prefill_reference_paged(q, kb, vb, table, sl, cu, max_len=most)
    o_c = ekv.attention_prefill_paged(q, kc, vc, table, sl, cu, max_len=most)
    assert same_bits(o_b, o_c)
    check(o_b, q, k, v, lens, klens)
    wide_b = ekv.attention_prefill_reference_paged(q, kb, vb, table, sl, cu)
    assert same_bits(wide_b, ekv.attention_prefill_paged(q, kc, vc, table, sl, cu))
    check(wide_b, q, k, v, lens, klens)
    plan = lambda keys: kernels.lib.exk_prefill_splits(sum(lens), len(lens), Hq, Hkv, keys, kernels.num_sms())  # noqa: E731
    if plan(-(-most // 16) * 16) == plan(sum(klens)) == 1:       # split on neither side: the same order of sums
        assert same_bits(o_b, ekv.attention_prefill(q, k, v, cu, ck))
    kernels.check_status()


@pytest.mark.gpu
def test_pages_outside_the_pool_read_as_zeros_and_are_reported():
    q, _, _ = inputs(20, 1, 8, 2, seed=31)
    k, v, kb, vb, kc, vc, table, sl = _pools([300], 2, seed=32)
    cu = offsets([20]).cuda()
    bad = table.clone()
    bad[0, 3], bad[0, 9] = -1, 1 << 20
    k0, v0 = k.clone(), v.clone()
    for p in (3, 9):
        k0[16 * p:16 * p + 16] = 0
        v0[16 * p:16 * p + 16] = 0
    for call, a, b in ((ekv.attention_prefill_reference_paged, kb, vb), (ekv.attention_prefill_paged, kc, vc)):
        out = call(q, a, b, bad, sl, cu)
        with pytest.raises(RuntimeError, match="outside the pool"):
            kernels.check_status()
        check(out, q, k0, v0, [20], [300])


@pytest.mark.gpu
def test_lengths_past_the_table_or_the_workspace_are_cut_and_reported():
    q, _, _ = inputs(5, 1, 8, 2, seed=33)
    k, v, kb, vb, kc, vc, table, sl = _pools([100, 64], 2, seed=34, max_extra=0)
    cu = offsets([3, 2]).cuda()
    long = torch.tensor([500, 64], dtype=torch.int32, device="cuda")
    for call, a, b, lens, kw in ((ekv.attention_prefill_reference_paged, kb, vb, long, {}),
                                 (ekv.attention_prefill_paged, kc, vc, long, {}),
                                 (ekv.attention_prefill_paged, kc, vc, sl, dict(max_len=64))):
        out = call(q, a, b, table, lens, cu, **kw)
        with pytest.raises(RuntimeError, match="length"):
            kernels.check_status()
        check(out[3:], q[3:], k[100:], v[100:], [2], [64])         # the other sequence is as it should be


@pytest.mark.gpu
@pytest.mark.parametrize("idle", [1, 40])
def test_sequences_without_queries_are_not_read(idle):
    """Sequences that bring no query may have any length and any pages: the others'
    results are the same and nothing is reported."""
    lens, klens = [5] + [0] * idle + [7], [40] + [100] * idle + [64]
    q, _, _ = inputs(12, 1, 8, 2, seed=35)
    k, v, kb, vb, kc, vc, table, sl = _pools(klens, 2, seed=36)
    cu = offsets(lens).cuda()
    table[1:-1], sl[1:-1] = -9, 1 << 20
    for call, a, b in ((ekv.attention_prefill_reference_paged, kb, vb), (ekv.attention_prefill_paged, kc, vc)):
        out = call(q, a, b, table, sl, cu, max_len=64)
        kernels.check_status()
        check(out[:5], q[:5], k[:40], v[:40], [5], [40])
        check(out[5:], q[5:], k[-64:], v[-64:], [7], [64])


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [0, 3])
def test_many_sequences(pad):
    """More sequences than a warp holds (the other way to map blocks), some empty,
    with rows before the first and after the last that belong to none."""
    lens = [(7 * i) % 41 for i in range(70)]
    klens = [n + (13 * i) % 150 for i, n in enumerate(lens)]
    Hq, Hkv, n = 8, 2, sum(lens)
    q, _, _ = inputs(n + 2 * pad, 1, Hq, Hkv, seed=90)
    _, k, v = inputs(1, sum(klens), Hq, Hkv, seed=91)
    hold = torch.full_like(q, 5.0)
    out = ekv.attention_prefill(q, k, v, offsets(lens).cuda() + pad, offsets(klens).cuda(), out=hold)
    check(out[pad:], q[pad:pad + n], k, v, lens, klens)
    assert (hold[:pad] == 5).all() and (hold[pad + n:] == 5).all()
    # a sequence by itself, where the plan may split its keys otherwise
    a = b = pad
    for i, (m, L) in enumerate(zip(lens, klens)):
        if m and L and i % 9 == 0:
            kk, vv = k[b - pad:b - pad + L], v[b - pad:b - pad + L]
            one = ekv.attention_prefill(q[a:a + m], kk, vv, offsets([m]).cuda(), offsets([L]).cuda())
            check(one, q[a:a + m], kk, vv, [m], [L])
        a, b = a + m, b + L
    kernels.check_status()


@pytest.mark.gpu
def test_pools_past_32_bit_offsets():
    """Pools of 2.7e9 values: the pages in use lie at their end."""
    Hq, Hkv, pages = 16, 8, 165_000
    lens = [300, 70]
    k = synthetic.make_kv(1, sum(lens), Hkv, seed=95, key=True)[0]
    v = synthetic.make_kv(1, sum(lens), Hkv, seed=96, key=False)[0]
    q, _, _ = inputs(sum(lens), 1, Hq, Hkv, seed=97)
    table = torch.full((2, 19), -1, dtype=torch.int32)
    table[0] = pages - 1 - torch.arange(19)
    table[1, :5] = pages - 40 + torch.arange(5)
    table, sl, cu = table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), offsets(lens).cuda()
    ident = torch.cat([torch.ones(400, 64), torch.zeros(400, 64)], 1).cuda()
    kb, vb = (torch.zeros(1, pages * 16, Hkv, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ekv.rope_append_reference_paged(q, k, v, ident, kb, vb, table, sl, cu)
    o = ekv.attention_prefill_reference_paged(q, kb, vb, table, sl, cu)
    check(o, q, k, v, lens, lens)
    del kb, vb
    kc, vc = (ekv.PagedCompressedKV(pages, Hkv, D, 2, reserve=0.001) for _ in range(2))
    ekv.rope_append_paged(q, k, v, ident, kc, vc, table, sl, cu)
    assert same_bits(ekv.attention_prefill_paged(q, kc, vc, table, sl, cu), o)
    kernels.check_status()


@pytest.mark.gpu
def test_captured_call_follows_lengths_on_the_device_and_shares_no_workspace():
    """Two captured calls with splits, replayed at the same time on two streams after
    their lengths changed, equal eager calls."""
    Hq, Hkv, most = 8, 2, 4096
    runs = []
    for i in range(2):
        q, k, v = inputs(16, most, Hq, Hkv, seed=40 + i)
        cu = offsets([7, 5]).cuda()
        ck = offsets([2000, 1500]).cuda()
        out = torch.zeros_like(q)
        ekv.attention_prefill(q, k, v, cu, ck, out=out)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ekv.attention_prefill(q, k, v, cu, ck, out=out)
        runs.append((q, k, v, cu, ck, out, g, torch.cuda.Stream()))
    for q, k, v, cu, ck, out, g, s in runs:
        cu.copy_(offsets([3, 12]))
        ck.copy_(offsets([100, 3996]))
        out.fill_(9)
    torch.cuda.synchronize()
    for _ in range(20):
        for q, k, v, cu, ck, out, g, s in runs:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for q, k, v, cu, ck, out, g, s in runs:
        want = ekv.attention_prefill(q, k, v, cu, ck, out=torch.full_like(q, 9))
        assert same_bits(out, want) and (out[15:] == 9).all()
        check(out, q[:15], k, v, [3, 12], [100, 3996])
    kernels.check_status()


@pytest.mark.gpu
def test_repeat_and_other_stream_give_the_same_bits():
    lens = [1000, 333]
    q, k, v = inputs(1333, 1333, 28, 4, seed=50)
    cu = offsets(lens).cuda()
    a = ekv.attention_prefill(q, k, v, cu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        outs = [ekv.attention_prefill(q, k, v, cu) for _ in range(10)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(same_bits(a, b) for b in outs)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,klens", [([300, 77, 1], [300, 77, 1]), ([5], [6000])])
def test_output_over_the_queries(lens, klens):
    """out = q: a block's queries are read before its rows are written (with splits,
    before the merge writes them)."""
    q, k, v = inputs(sum(lens), sum(klens), 8, 2, seed=100)
    cu, ck = offsets(lens).cuda(), offsets(klens).cuda()
    want = ekv.attention_prefill(q, k, v, cu, ck)
    own = q.clone()
    assert ekv.attention_prefill(own, k, v, cu, ck, out=own) is own
    assert same_bits(own, want)


@pytest.mark.gpu
@pytest.mark.parametrize("one_stream", [True, False])
def test_calls_from_two_threads(one_stream):
    """Two threads that call at once, on one stream or on their own: every call has its
    own workspace, so each result is what the call alone gives."""
    import threading
    work = []
    for i in range(2):
        q, k, v = inputs(12, 5000, 8, 2, seed=110 + i)
        kk, vv, kb, vb, kc, vc, table, sl = _pools([700, 333], 2, seed=120 + i)
        cu, ck = offsets([12]).cuda(), offsets([5000]).cuda()
        q2, _, _ = inputs(30, 1, 8, 2, seed=130 + i)
        c2 = offsets([20, 10]).cuda()
        want = (ekv.attention_prefill(q, k, v, cu, ck), ekv.attention_prefill_paged(q2, kc, vc, table, sl, c2))
        work.append(((q, k, v, cu, ck), (q2, kc, vc, table, sl, c2), want, []))
    torch.cuda.synchronize()
    shared = torch.cuda.Stream()

    def run(args, pargs, want, bad):
        with torch.cuda.stream(shared if one_stream else torch.cuda.Stream()):
            for _ in range(60):
                a, b = ekv.attention_prefill(*args), ekv.attention_prefill_paged(*pargs)
                if not (same_bits(a, want[0]) and same_bits(b, want[1])):
                    bad.append(1)

    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not any(w[3] for w in work)
    kernels.check_status()


@pytest.mark.gpu
def test_prefill_of_one_token_agrees_with_decode_attention():
    """One query per sequence: the decode kernel's result within both bounds."""
    Hq, Hkv, klens = 32, 8, [1000, 513, 260]
    q, _, _ = inputs(3, 1, Hq, Hkv, seed=60)
    k, v, kb, vb, kc, vc, table, sl = _pools(klens, Hkv, seed=61)
    one = ekv.attention_prefill_paged(q, kc, vc, table, sl, offsets([1, 1, 1]).cuda())
    dec = kernels.attention_paged(q, kc, vc, table, sl)
    o, tol = reference(q, k, v, [1, 1, 1], klens)
    assert ((one.double().cpu() - dec.double().cpu()).abs() <= 2 * tol).all()
    check(one, q, k, v, [1, 1, 1], klens)


@pytest.mark.gpu
def test_prefill_of_nothing():
    q, k, v = inputs(4, 4, 8, 2, seed=70)
    cu = torch.zeros(3, dtype=torch.int32, device="cuda")
    out = ekv.attention_prefill(q[:0], k, v, cu, cu)
    assert out.shape == (0, 8, D)
    hold = torch.full_like(q, 3)
    ekv.attention_prefill(q, k, v, cu, cu, out=hold)            # rows of no sequence
    assert (hold == 3).all()


def test_refusals():
    """Arguments that do not fit are refused on the host, before any launch."""
    q = torch.zeros(4, 8, D, dtype=torch.bfloat16)
    k = torch.zeros(4, 2, D, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    for args in ((q, k, k, cu), (q.float(), k, k, cu)):
        with pytest.raises(ValueError):
            ekv.attention_prefill(*args)
    table = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError):
        ekv.attention_prefill_reference_paged(q, k[None], k[None], table, cu[1:], cu)
    with pytest.raises(ValueError):
        ekv.attention_prefill_reference_paged(q, k.view(1, 4, 2, D), k.view(1, 4, 2, D), table, cu[1:], cu, max_len=65)


@pytest.mark.gpu
def test_refusals_on_device_tensors():
    q, k, v = inputs(8, 8, 8, 2, seed=80)
    cu = offsets([8]).cuda()
    wrong = [
        (q, k[:, :, :64], v, cu), (q, k.float(), v, cu), (q[:, :7], k, v, cu), (q, k, v[:7], cu),
        (q, k, v, cu.long()), (q, k, v, cu.cpu()), (q[..., ::2], k, v, cu), (q, k[:7], v[:7], cu),
    ]
    for args in wrong:
        with pytest.raises((ValueError, RuntimeError)):
            ekv.attention_prefill(*args)
    with pytest.raises(RuntimeError, match="16 query heads"):
        ekv.attention_prefill(q.view(4, 16, D).repeat(1, 2, 1)[:, :17].contiguous(), k[:4, :1].contiguous(),
                              v[:4, :1].contiguous(), offsets([4]).cuda())
    odd = torch.zeros(8 * 8 * D + 4, dtype=torch.bfloat16, device="cuda")[4:].view(8, 8, D)
    with pytest.raises(ValueError, match="16-byte"):
        ekv.attention_prefill(odd, k, v, cu)
