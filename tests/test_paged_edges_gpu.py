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
