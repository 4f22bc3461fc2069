"""KV caches behind the reference's cache interface (exactkv/cache.py: prefill_slot,
append, T, nbytes, buffers, kernel_args, check_overflow), built around a token
count that lives on the device.

Buffers (the format the kernels read; include/exactkv_b200.h):
  sm, code   u8  [B, TS, H, 128] / [B, TS, H, 64]
  base       u8  [B, TS/16, H, 128]
  rowmask    i32 [B, TS/16, H]        bit r: token r of the page is a raw row
  rowoff     i32 [B, TS/16, H]        pool row of the page's first raw row
  raw        bf16 [cap + B*H*16, 128] pool rows [0, cnt) for encoded pages,
                                      then one 16-row open page per (sequence, head)

The newest, partly filled page of every sequence lives in its open-page rows and
is marked all-raw (rowmask 0xFFFF, rowoff at those rows), so attention reads it
like any other page; when it fills, the device append kernel encodes it in place
and opens the next one (exk_append_token).

Pool policy, this package's own: every append goes through that device kernel,
and at each page boundary the host makes one check (check_overflow(), one sync
for all caches) that keeps at least one worst-case page (every row raw, B*H*16
rows) free in every pool. So an append can never overflow and no page is ever
encoded twice. Only a prefill, whose raw rows have no useful bound, can
overflow: its pages are then encoded again into a grown pool.
"""
import torch

from . import kernels
from ._lib import CView
from .kernels import P

_GROW_ALIGN = 256   # pool capacities are multiples of this many rows


class RawPool:
    """The raw bf16 rows of one cache: `cap` slots for encoded pages followed by
    the open-page area of `nseq` x `H` pages of 16 rows."""

    def __init__(self, nseq, H, D, cap, device):
        self.nseq, self.H, self.D, self.device = nseq, H, D, device
        self.cap = cap
        self.rows = torch.zeros(cap + nseq * H * P, D, dtype=torch.bfloat16, device=device)
        self.moves = 0

    def open_pages(self):
        """The open-page area as [nseq, H, 16, D]."""
        return self.rows[self.cap:].view(self.nseq, self.H, P, self.D)

    def open_page_rows(self):
        """int32 [nseq, H]: pool row of each open page's first row."""
        first = self.cap + P * torch.arange(self.nseq * self.H, dtype=torch.int32, device=self.device)
        return first.view(self.nseq, self.H)

    def enlarge(self, used, need):
        """Re-allocates with room for at least `need` slots, keeping slots [0, used)
        and the open pages. Capacity grows by half at least, so a cache that keeps
        overflowing pays a logarithmic number of copies."""
        cap = max(need, self.cap + self.cap // 2)
        cap = -(-cap // _GROW_ALIGN) * _GROW_ALIGN
        rows = torch.empty(cap + self.nseq * self.H * P, self.D, dtype=torch.bfloat16, device=self.device)
        if used:
            rows[:used].copy_(self.rows[:used])
        rows[cap:].copy_(self.rows[self.cap:])
        self.rows, self.cap = rows, cap
        self.moves += 1


class CompressedKV:
    """One layer's keys (or values) for B sequences of up to TS tokens, H KV heads,
    head dim 128. `reserve`: initial pool slots as a fraction of all rows."""

    def __init__(self, B, TS, H, D, device="cuda", reserve=0.01):
        if TS % P != 0 or D != 128:
            raise ValueError("TS must be a multiple of 16 and D = 128 (Qwen2/2.5/3, Llama-3 family)")
        self.B, self.TS, self.H, self.D = B, TS, H, D
        self.dev = torch.device(device)
        u8 = dict(dtype=torch.uint8, device=self.dev)
        i32 = dict(dtype=torch.int32, device=self.dev)
        npages = TS // P
        self.sm = torch.zeros(B, TS, H, D, **u8)
        self.code = torch.zeros(B, TS, H, D // 2, **u8)
        self.base = torch.zeros(B, npages, H, D, **u8)
        self.rowmask = torch.zeros(B, npages, H, **i32)
        self.rowoff = torch.zeros(B, npages, H, **i32)
        self.cnt = torch.zeros(1, **i32)                 # pool slots taken by encoded pages
        self.pool = RawPool(B, H, D, max(64, int(B * TS * H * reserve)), self.dev)
        self.lens = [0] * B                              # tokens per sequence
        self.T = 0                                       # tokens of the batch (the last prefilled slot's, as the reference)
        self._t_dev = torch.zeros(1, **i32)              # T on the device, for the append kernel
        self._t_dev_stale = False                        # T moved by device-length steps
        self._checked = True                             # headroom verified since the last page boundary
        self._bind()

    # ------------------------------------------------------------------ views
    @property
    def raw(self):
        return self.pool.rows

    @property
    def cap(self):
        return self.pool.cap

    @property
    def grows(self):
        return self.pool.moves

    def _bind(self):
        """Descriptors that name the pool's storage; rebuilt when it moves."""
        self._kargs = (self.sm, self.code, self.base, self.rowmask, self.rowoff, self.pool.rows.view(torch.int16))
        self._view = CView(self.sm.data_ptr(), self.code.data_ptr(), self.base.data_ptr(), self.rowmask.data_ptr(),
                           self.rowoff.data_ptr(), self.pool.rows.data_ptr(), self.pool.rows.shape[0])

    def kernel_args(self):
        return self._kargs

    def kernel_view(self):
        return self._view

    def tail_offsets(self):
        return self.pool.open_page_rows()

    def encoder_buffers(self):
        """The dict kernels.encode_pages writes into."""
        return dict(sm=self.sm, code=self.code, base=self.base, rowmask=self.rowmask, rowoff=self.rowoff,
                    raw=self.pool.rows, cnt=self.cnt, cap=self.pool.cap, TS=self.TS, H=self.H, D=self.D)

    def buffers(self):
        return dict(shape=(self.B, self.TS, self.H, self.D), sm=self.sm, code=self.code, base=self.base,
                    rowmask=self.rowmask, rowoff=self.rowoff, raw=self.pool.rows)

    def nbytes(self):
        return sum(t.numel() * t.element_size()
                   for t in (self.sm, self.code, self.base, self.rowmask, self.rowoff, self.pool.rows))

    # ------------------------------------------------------------------ pool
    def _relocate(self, used, need):
        """Moves the pool (keeping slots [0, used)) and re-points every open page."""
        self.pool.enlarge(used, need)
        self._bind()
        first = self.pool.open_page_rows()
        for b, t in enumerate(self.lens):
            if t < self.TS:
                self.rowoff[b, t // P] = first[b]

    def headroom_rows(self, pages=1):
        """Slots that `pages` pages of the whole batch need when every row is raw."""
        return pages * self.B * self.H * P

    def ensure_headroom(self, pages):
        """Before `pages` more pages are appended: one sync to read the slot counter,
        then grow so that even `pages` pages of nothing but raw rows fit. Returns
        True when the pool moved (work enqueued with the old buffers, such as a
        captured graph, must be rebuilt)."""
        return self._make_room(int(self.cnt.item()), pages)

    def _make_room(self, used, pages):
        need = used + self.headroom_rows(pages)
        self._checked = True
        if need <= self.pool.cap:
            return False
        # a quarter window of slack: the next check, after `pages` pages that
        # escaped a few per cent of their rows as usual, must not find the pool
        # short again (each growth moves the pool and invalidates captured work)
        self._relocate(used, need + self.headroom_rows(pages) // 4)
        return True

    # ------------------------------------------------------------------ filling
    def prefill_slot(self, b, x):
        """x: [1, T, H, D] bf16 (any strides, channels contiguous) for sequence slot b.
        Full pages are encoded (raw-pool slots follow the slot order of the calls);
        the rest goes to the slot's open page. Syncs once (the pool counter) and,
        if the pool overflowed, encodes the slot's pages again into a larger pool."""
        T = x.shape[1]
        if not 0 < T <= self.TS:
            raise ValueError(f"prefill of {T} tokens into a cache of {self.TS}")
        npg = T // P
        if npg:
            strides = (x.stride(0), P * x.stride(1), x.stride(1), x.stride(2))
            start = self.cnt.clone()
            kernels.encode_pages(x, strides, self.encoder_buffers(), b, 0, 1, npg)
            used = int(self.cnt.item())
            if used > self.pool.cap:
                self._relocate(int(start.item()), used)
                self.cnt.copy_(start)
                kernels.encode_pages(x, strides, self.encoder_buffers(), b, 0, 1, npg)
                if int(self.cnt.item()) > self.pool.cap:
                    raise RuntimeError("raw pool still too small after growing")
        self.lens[b] = T
        if npg < self.TS // P:
            self.rowmask[b, npg] = (1 << P) - 1
            self.rowoff[b, npg] = self.pool.open_page_rows()[b]
            self.pool.open_pages()[b, :, : T - npg * P] = x[0, npg * P:].transpose(0, 1)
        self.T = T
        self._t_dev.fill_(T)
        self._t_dev_stale = False
        self._checked = False

    def append(self, x):
        """x: [B, H, D] bf16, one new token per sequence (every sequence at the
        same length T). The device append kernel writes it and, when the page
        fills, encodes the page and opens the next. A boundary that the host has
        not checked since the previous one is checked here first."""
        if any(t != self.T for t in self.lens):
            raise RuntimeError("append needs every sequence at the same length (use append_dev for varlen)")
        if self.T >= self.TS:
            raise RuntimeError("cache full")
        if self.T % P == P - 1 and not self._checked:
            self.ensure_headroom(1)
        if self._t_dev_stale:                            # device-length steps moved T since
            self._t_dev.fill_(self.T)
            self._t_dev_stale = False
        kernels.append_token(x, self, self._t_dev)
        kernels.advance_length(self._t_dev, 1)
        self._count(1)
        if self.T % P == 0:
            self._checked = False

    # ------------------------------------------------------------------ device-length steps
    def append_dev(self, x, T_dev):
        """Enqueues the append of one token per sequence at the device-side length
        *T_dev (no host bookkeeping; see kernels.append_token). The host's count
        is advanced with note_appended() once the step is enqueued."""
        kernels.append_token(x, self, T_dev)

    def note_appended(self, n=1):
        """Records n tokens appended by device-length steps (append_dev)."""
        self._count(n)
        self._t_dev_stale = True

    def _count(self, n):
        self.T += n
        self.lens = [t + n for t in self.lens]

    def lengths(self):
        """The sequences' token counts as a device int32 tensor (the T_dev of a
        variable-length batch for the device-length calls)."""
        return torch.tensor(self.lens, dtype=torch.int32, device=self.dev)


class PagedCompressedKV:
    """A pool of `pages` 16-token pages of one layer's keys (or values) in the
    compressed format, H KV heads, head dim 128, for up to `max_seqs` sequences
    that are being written: each has a tail slot, where its open page is kept
    raw. Written by kernels.rope_append_paged, read by kernels.attention_paged
    and kernels.attention_prefill_paged, all through int32 block tables that the
    caller keeps. `reserve`: initial raw-pool slots as a fraction of all rows."""

    def __init__(self, pages, H, D, max_seqs, device="cuda", reserve=0.01):
        if pages <= 0 or max_seqs <= 0 or H <= 0 or D != 128:
            raise ValueError("pages, H and max_seqs must be positive and D = 128 (Qwen2/2.5/3, Llama-3 family)")
        self.B, self.TS, self.H, self.D = 1, pages * P, H, D       # the pages as one long sequence of rows
        self.dev = torch.device(device)
        u8 = dict(dtype=torch.uint8, device=self.dev)
        i32 = dict(dtype=torch.int32, device=self.dev)
        self.sm = torch.zeros(1, pages * P, H, D, **u8)
        self.code = torch.zeros(1, pages * P, H, D // 2, **u8)
        self.base = torch.zeros(1, pages, H, D, **u8)
        self.rowmask = torch.zeros(1, pages, H, **i32)
        self.rowoff = torch.zeros(1, pages, H, **i32)
        self.cnt = torch.zeros(1, **i32)
        self.pool = RawPool(max_seqs, H, D, max(64, int(pages * P * H * reserve)), self.dev)
        self._bind()

    @property
    def raw(self):
        return self.pool.rows

    @property
    def cap(self):
        return self.pool.cap

    def _bind(self):
        self._view = CView(self.sm.data_ptr(), self.code.data_ptr(), self.base.data_ptr(), self.rowmask.data_ptr(),
                           self.rowoff.data_ptr(), self.pool.rows.data_ptr(), self.pool.rows.shape[0])

    def kernel_view(self):
        return self._view

    def buffers(self):
        return dict(shape=(1, self.TS, self.H, self.D), sm=self.sm, code=self.code, base=self.base,
                    rowmask=self.rowmask, rowoff=self.rowoff, raw=self.pool.rows, cnt=self.cnt, cap=self.pool.cap)

    def nbytes(self):
        return sum(t.numel() * t.element_size()
                   for t in (self.sm, self.code, self.base, self.rowmask, self.rowoff, self.pool.rows))

    def ensure_headroom(self, tokens):
        """Before `tokens` more tokens are appended: one sync to read the slot counter,
        then grow so that even `tokens` tokens of nothing but raw rows fit (they and
        the rows already in open pages: 16 for each sequence). Returns True when the
        pool moved (a captured graph must be captured again). Raises RuntimeError when
        appends have wanted more raw rows than there were: the pages that had no room
        are lost (readers report them) and their sequences must be appended again
        (after compact() without them).

        The reservation is for the worst case, the size of the tokens uncompressed: a long
        prompt appended in chunks, each after a call of its own, needs less."""
        return self._grow(int(self.cnt.item()), (tokens + P * self.pool.nseq) * self.H)

    def compact(self, block_table):
        """Gives the raw rows of pages that no sequence uses any more back to the pool:
        appends only ever take new ones, so a pool whose pages pass from sequence to
        sequence runs full without it. block_table: int32, any shape, the pages in use
        (others' contents are lost; entries outside the pool, such as -1, are passed
        over). Their raw rows move to the front of the pool, whose storage stays where
        it is: a captured graph stays valid. Syncs. Returns the rows in use."""
        at = block_table.to(self.rowoff.device).flatten().long()
        pages = torch.unique(at[(at >= 0) & (at < self.TS // P)])
        first = self.rowoff[0, pages].long()                         # [pages in use, H]
        kept = (first >= 0) & (first < self.pool.cap)                # not open, and not without room
        rows = (self.rowmask[0, pages, :, None] >> torch.arange(P, device=pages.device) & 1).sum(-1) * kept
        end = rows.flatten().cumsum(0).view_as(rows)
        total = int(end[-1, -1]) if len(pages) else 0
        src = torch.repeat_interleave((first - end + rows).flatten(), rows.flatten(), output_size=total)
        self.pool.rows[:total] = self.pool.rows[src + torch.arange(total, device=pages.device)]
        self.rowoff[0, pages] = torch.where(kept, end - rows, first).int()
        # (a page that a table names before its sequence comes to it must not claim, at a
        # later call, the slots that its old rows had)
        gone = torch.ones(self.TS // P, 1, dtype=torch.bool, device=pages.device)
        gone[pages] = False
        self.rowmask[0].masked_fill_(gone, 0)
        self.cnt.fill_(total)
        return total

    def _make_room(self, used, pages):
        """check_overflow()'s share: room for `pages` worst-case pages of every sequence."""
        return self._grow(used, pages * P * self.pool.nseq * self.H)

    def _grow(self, used, rows):
        need, old = used + rows, self.pool.cap
        if used > old:
            raise RuntimeError(f"{used} raw rows appended to a pool of {old}: pages without room were not kept")
        if need <= old:
            return False
        self.pool.enlarge(used, need)
        self._bind()
        # entries at or past the old capacity are open pages': they move with the tail slots
        self.rowoff += (self.rowoff >= old).int() * (self.pool.cap - old)
        return True


class BF16KV:
    """Uncompressed bf16 cache [B, TS, H, D] with the same interface."""

    def __init__(self, B, TS, H, D, device="cuda"):
        self.buf = torch.zeros(B, TS, H, D, dtype=torch.bfloat16, device=device)
        self.T = 0
        self.cnt = None

    def prefill_slot(self, b, x):
        T = x.shape[1]
        self.buf[b, :T].copy_(x[0])
        self.T = T

    def append(self, x):
        self.buf[:, self.T].copy_(x)
        self.T += 1

    def nbytes(self):
        return self.buf.numel() * self.buf.element_size()


def check_overflow(caches):
    """The host check after a page boundary: one sync reads the slot counters of
    all compressed caches (and the kernels' status word, raising on a fault), then
    every pool with less than one worst-case page a sequence free grows. Returns the
    number of caches that grew. A PagedCompressedKV, whose lengths the host does not
    know, is looked at in every call: one call in 16 steps of a token each is enough."""
    cs = [c for c in caches if isinstance(c, PagedCompressedKV) or isinstance(c, CompressedKV) and not c._checked]
    if not cs:
        return 0
    status = kernels.status_tensor(cs[0].dev)
    vals = torch.cat([c.cnt for c in cs] + [status]).tolist()
    if vals[-1] != 0:
        kernels.check_status(cs[0].dev)
    return sum(int(c._make_room(used, 1)) for c, used in zip(cs, vals[:-1]))
