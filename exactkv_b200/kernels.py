"""Drop-in replacement of the reference's exactkv/kernels.py, backed by the
sm_100a kernels of libexactkv_b200.so through its C ABI.

Same public names and argument meanings as the reference module
(exactkv/kernels.py:273-346): P, LOG2E, choose_split, attention_compressed,
attention_reference, decode_to_bf16, encode_pages. Everything runs on the
caller's current CUDA stream and nothing synchronises the host, except
check_status(). There is no CPU or Triton fallback: without the library this
module fails to import.

Differences from the reference, all invisible to callers of the reference API:
  * the split layout comes from call_plan() (persistent CTAs over the SMs:
    equal-length splits, or one equal run of pages per CTA when that balances
    better) instead of choose_split(); choose_split() is kept for compatibility;
  * BLOCK_N and num_stages are accepted and ignored (pages are 16 tokens and
    the TMA ring depth is fixed); num_warps selects 4 or 8 consumer warps
    (default 8) — the compressed and bf16 kernels called with the same value
    stay bit-identical, as in the reference;
  * the page encoder assigns raw-pool slots in (sequence, page, head) order,
    so rowoff/raw match encode_reference byte for byte as well.
"""
import ctypes

import torch

from ._lib import APPEND, CVIEW, PREFILL, CView, Partials, check, lib

LOG2E = 1.4426950408889634
P = 16          # tokens per page
D = 128         # head dimension

_I32 = ctypes.c_int32


def choose_split(B, Hkv, T, BLOCK_N, target=512):
    """The reference's split rule (exactkv/kernels.py:273-277): at most `target`
    programs, split length a multiple of BLOCK_N. Returns (splits, split length)."""
    def cdiv(a, b):
        return (a + b - 1) // b

    ns = max(1, min(cdiv(T, BLOCK_N), target // max(1, B * Hkv)))
    split_len = cdiv(cdiv(T, ns), BLOCK_N) * BLOCK_N
    return cdiv(T, split_len), split_len


_SMS = {}


def num_sms(device=None):
    """SM count of a CUDA device (the number of persistent attention CTAs)."""
    dev = _device_index(device)
    if dev not in _SMS:
        n = lib.exk_num_sms(dev)
        if n <= 0:
            check(n if n < 0 else -1, "exk_num_sms")
        _SMS[dev] = n
    return _SMS[dev]


def plan_splits(B, Hkv, T, device=None, num_ctas=None):
    """(splits, split length in tokens) of the attention plan."""
    ns, sl = _I32(), _I32()
    ctas = num_ctas if num_ctas is not None else num_sms(device)
    check(lib.exk_plan_splits(B, Hkv, T, ctas, ctypes.byref(ns), ctypes.byref(sl)), "exk_plan_splits")
    return ns.value, sl.value


def call_plan(B, Hkv, T, device=None, num_warps=None, num_ctas=None, any_length=False):
    """(splits, split length) for one whole decode-attention call with host-side T:
    the balanced plan (split length 0: every CTA gets an equal run of the call's
    pages across sequence boundaries; exk_plan_balanced) when it is estimated
    faster than the uniform plan of plan_splits(), else the uniform one. The
    compressed and bf16 calls with the same arguments get the same plan.
    any_length: the plan of a device-length call with one length for the batch
    and capacity T (the balanced plan's kernel cuts the length it reads)."""
    ns = _I32()
    ctas = num_ctas if num_ctas is not None else num_sms(device)
    check(lib.exk_plan_balanced(B, Hkv, T, ctas, _consumer_warps(num_warps), int(bool(any_length)),
                                ctypes.byref(ns)), "exk_plan_balanced")
    if ns.value > 0:
        return ns.value, 0
    return plan_splits(B, Hkv, T, device, num_ctas)


def _device_index(device):
    if device is None:
        return torch.cuda.current_device()
    if isinstance(device, int):
        return device
    device = torch.device(device)
    return device.index if device.index is not None else torch.cuda.current_device()


# ----------------------------------------------------------------------------- status word and scratch

_STATUS = {}   # device index -> int32[1] status word written by the kernels


def status_tensor(device):
    dev = _device_index(device)
    t = _STATUS.get(dev)
    if t is None:
        t = _STATUS[dev] = torch.zeros(1, dtype=torch.int32, device=f"cuda:{dev}")
    return t


def check_status(device=None, reset=True):
    """Synchronises with the device and raises RuntimeError if a kernel recorded a
    fault (a timed-out wait or an out-of-range raw index) since the last check."""
    t = status_tensor(device)
    code = int(t.item())
    if code != 0:
        if reset:
            t.zero_()
        raise RuntimeError(f"exactkv_b200 device status {code}: {lib.exk_status_string(code).decode()}")
    return 0


# ----------------------------------------------------------------------------- split workspaces

_WS = {}  # (device, stream, rows, ns) -> (o, m, l, Partials); reused by calls on the same stream


def _workspace(device, stream, rows, ns, split_len, heads=0):
    """Split partials o [rows, ns, 128], m, l [rows, ns], for a plan of ns splits
    of split_len tokens and `heads` KV heads per work item (0: the default)."""
    key = (device.index, stream, rows, ns)
    ws = _WS.get(key)
    if ws is None:
        f32 = dict(device=device, dtype=torch.float32)
        o, m, l = torch.empty(rows, ns, D, **f32), torch.empty(rows, ns, **f32), torch.empty(rows, ns, **f32)
        ws = _WS[key] = (o, m, l, Partials(o.data_ptr(), m.data_ptr(), l.data_ptr(), ns, split_len))
    ws[3].split_len = split_len
    ws[3].heads = heads
    return ws


def _consumer_warps(num_warps):
    return 4 if num_warps is not None and num_warps <= 4 else 8


def _view_from_dict(c):
    raw = c["raw"]
    cv = CView(c["sm"].data_ptr(), c["code"].data_ptr(), c["base"].data_ptr(), c["rowmask"].data_ptr(),
               c["rowoff"].data_ptr(), raw.data_ptr(), raw.shape[0])
    return cv, c["shape"][1], c["shape"][2]


_ARGS_VIEWS = {}  # id(kernel_args() tuple) -> (the tuple, its exk_cview)


def _view_from_args(kargs):
    """exk_cview of a kernel_args() tuple (sm, code, base, rowmask, rowoff, raw as
    int16 [rows, 128]), the form a reference CompressedKV hands its kernels
    (exactkv/cache.py:39-47). A cache rebuilds that tuple only when its raw pool
    grows, so the view is kept per tuple object."""
    hit = _ARGS_VIEWS.get(id(kargs))
    if hit is not None and hit[0] is kargs:
        return hit[1]
    sm, code, base, rowmask, rowoff, raw = kargs
    cv = CView(sm.data_ptr(), code.data_ptr(), base.data_ptr(), rowmask.data_ptr(), rowoff.data_ptr(),
               raw.data_ptr(), raw.shape[0])
    if len(_ARGS_VIEWS) > 256:
        _ARGS_VIEWS.clear()
    _ARGS_VIEWS[id(kargs)] = (kargs, cv)
    return cv


def _cache_args(c):
    """(exk_cview, TS, Hkv) from a cache object or from its .buffers() dict, as the
    reference's _cache_args takes them (exactkv/kernels.py:302-307): this package's
    CompressedKV (its view is kept on the cache), or any cache with the reference's
    kernel_args() / .TS / .H, the reference's own CompressedKV included."""
    if isinstance(c, dict):
        return _view_from_dict(c)
    view = getattr(c, "kernel_view", None)
    if view is not None:
        return view(), c.TS, c.H
    return _view_from_args(c.kernel_args()), c.TS, c.H


def _check_q(q, T, TS):
    if q.dim() != 3 or q.shape[2] != D or q.dtype != torch.bfloat16 or not q.is_contiguous() or not q.is_cuda:
        raise ValueError("q must be a contiguous CUDA bf16 tensor [B, Hq, 128]")
    if not 0 < T <= TS:
        raise ValueError(f"T={T} out of range (1..{TS})")


def _check_out(out, q):
    """An output for q's shape: a CUDA tensor, or pinned host memory that the merge
    kernel writes directly (a zero-copy device-to-host result)."""
    if out.shape != q.shape or out.dtype != torch.bfloat16 or not out.is_contiguous():
        raise ValueError("out must be a contiguous bf16 tensor shaped like q")
    if not out.is_cuda and not out.is_pinned():
        raise ValueError("out must be a CUDA tensor or pinned host memory")
    return out


def attention_split(q, kc, vc, T, ws, s0, s1, num_warps=None):
    """Split partials of the compressed attention for splits [s0, s1) of ws's plan
    (the per-GPU step of a KV-sequence split). ws: (o, m, l, Partials)."""
    ka, TS, Hkv = _cache_args(kc)
    va, _, _ = _cache_args(vc)
    _check_q(q, T, TS)
    B, Hq, _ = q.shape
    dev = q.device.index
    stream = torch.cuda.current_stream(q.device).cuda_stream
    rc = lib.exk_attn_split_compressed(q.data_ptr(), ctypes.byref(ka), ctypes.byref(va), B, TS, Hkv, Hq, T, s0, s1,
                                       ctypes.byref(ws[3]), _consumer_warps(num_warps), D ** -0.5 * LOG2E,
                                       status_tensor(dev).data_ptr(), dev, stream)
    check(rc, "exk_attn_split_compressed")


def attention_split_bf16(q, k, v, T, ws, s0, s1, num_warps=None):
    """attention_split on uncompressed bf16 K, V [B, TS, Hkv, 128] (contiguous):
    the same partials as the compressed kernel for the same values and plan."""
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16 or not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("k and v must be contiguous bf16 [B, TS, Hkv, 128]")
    TS, Hkv = k.shape[1], k.shape[2]
    _check_q(q, T, TS)
    B, Hq, _ = q.shape
    dev = q.device.index
    stream = torch.cuda.current_stream(q.device).cuda_stream
    rc = lib.exk_attn_split_bf16(q.data_ptr(), k.data_ptr(), v.data_ptr(), B, TS, Hkv, Hq, T, s0, s1,
                                 ctypes.byref(ws[3]), _consumer_warps(num_warps), D ** -0.5 * LOG2E,
                                 status_tensor(dev).data_ptr(), dev, stream)
    check(rc, "exk_attn_split_bf16")


def merge_partials(ws, rows, out):
    """Merge of the workspace's splits into bf16 out [rows, 128] (a CUDA tensor or
    pinned host memory), on the workspace device's current stream."""
    dev = ws[0].device
    stream = torch.cuda.current_stream(dev).cuda_stream
    check(lib.exk_attn_merge(ctypes.byref(ws[3]), rows, out.data_ptr(), dev.index, stream), "exk_attn_merge")
    return out


def attention_compressed(q, kc, vc, T, BLOCK_N=64, num_warps=None, num_stages=1):
    """q [B, Hq, D] bf16 contiguous; kc, vc: CompressedKV objects (or their .buffers()
    dicts); T: valid tokens. Returns bf16 [B, Hq, D]. Bit-identical to
    attention_reference called with the same num_warps."""
    ka, TS, Hkv = _cache_args(kc)
    va, _, _ = _cache_args(vc)
    _check_q(q, T, TS)
    B, Hq, _ = q.shape
    dev = q.device.index
    stream = torch.cuda.current_stream(q.device).cuda_stream
    ns, sl = call_plan(B, Hkv, T, dev, num_warps)
    ws = _workspace(q.device, stream, B * Hq, ns, sl)
    out = torch.empty_like(q)
    rc = lib.exk_attention_compressed(q.data_ptr(), ctypes.byref(ka), ctypes.byref(va), B, TS, Hkv, Hq, T,
                                      ctypes.byref(ws[3]), out.data_ptr(), _consumer_warps(num_warps),
                                      D ** -0.5 * LOG2E, status_tensor(dev).data_ptr(), dev, stream)
    check(rc, "exk_attention_compressed")
    return out


def attention_reference(q, k, v, T, BLOCK_N=64, num_warps=None, num_stages=1):
    """The same computation on uncompressed bf16 K, V of shape [B, TS, Hkv, D] (contiguous)."""
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16 or not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("k and v must be contiguous bf16 [B, TS, Hkv, 128]")
    TS, Hkv = k.shape[1], k.shape[2]
    _check_q(q, T, TS)
    B, Hq, _ = q.shape
    dev = q.device.index
    stream = torch.cuda.current_stream(q.device).cuda_stream
    ns, sl = call_plan(B, Hkv, T, dev, num_warps)
    ws = _workspace(q.device, stream, B * Hq, ns, sl)
    out = torch.empty_like(q)
    rc = lib.exk_attention_bf16(q.data_ptr(), k.data_ptr(), v.data_ptr(), B, TS, Hkv, Hq, T, ctypes.byref(ws[3]),
                                out.data_ptr(), _consumer_warps(num_warps), D ** -0.5 * LOG2E,
                                status_tensor(dev).data_ptr(), dev, stream)
    check(rc, "exk_attention_bf16")
    return out


def decode_to_bf16(c, T):
    """Compressed buffers (a .buffers() dict) -> bf16 [B, T, H, D] through the same
    decoder the attention kernel uses."""
    cv, TS, H = _view_from_dict(c)
    B = c["shape"][0]
    dev = c["sm"].device
    out = torch.empty(B, T, H, D, dtype=torch.bfloat16, device=dev)
    stream = torch.cuda.current_stream(dev).cuda_stream
    check(lib.exk_decode_to_bf16(ctypes.byref(cv), B, TS, H, T, out.data_ptr(),
                                 status_tensor(dev.index).data_ptr(), dev.index, stream), "exk_decode_to_bf16")
    return out


def encode_pages(src, strides, buf, b0, pg0, nb, npg):
    """Encode nb sequences x npg pages. src points at sequence b0's first page to
    encode; strides = (seq, page, token, head) in elements. buf: dict with sm, code,
    base, rowmask, rowoff, raw, cnt, cap, TS, H, D."""
    if buf["D"] != D or src.dtype != torch.bfloat16 or src.stride(-1) != 1:
        raise ValueError("src must be bf16 with contiguous channels; D = 128 only")
    dev = src.device
    stream = torch.cuda.current_stream(dev).cuda_stream
    s_b, s_pg, s_p, s_h = (int(s) for s in strides)
    rc = lib.exk_encode_pages(src.data_ptr(), s_b, s_pg, s_p, s_h, buf["sm"].data_ptr(), buf["code"].data_ptr(),
                              buf["base"].data_ptr(), buf["rowmask"].data_ptr(), buf["rowoff"].data_ptr(),
                              buf["raw"].data_ptr(), int(buf["cap"]), buf["cnt"].data_ptr(),
                              b0, pg0, nb, npg, buf["H"], buf["TS"], status_tensor(dev.index).data_ptr(),
                              dev.index, stream)
    check(rc, "exk_encode_pages")


# ----------------------------------------------------------------------------- device-length decode steps
#
# One decode step whose token count lives on the device (an int32 tensor, the
# tokens held before the step), so the whole step can be enqueued once and
# replayed (CUDA graphs): append_token writes and, at page boundaries, encodes;
# attention_compressed_devlen reads T from the device with the plan for the
# caches' capacity; advance_length moves the count on. No host synchronisation.

def _stride_of(T_dev, B):
    """0: one length for the batch (a 1-element tensor); 1: one per sequence."""
    if T_dev.dtype != torch.int32 or not T_dev.is_contiguous() or T_dev.numel() not in (1, B):
        raise ValueError("T_dev must be a contiguous int32 tensor of 1 or B lengths")
    return 0 if T_dev.numel() == 1 else 1


def devlen_plan(B, Hkv, TS, T_dev, device=None, num_warps=None):
    """(splits, split length) of a device-length call over caches of capacity
    TS: with one length for the batch the balanced plan where it is estimated
    faster (call_plan(any_length=True)), else plan_splits() for the capacity."""
    if _stride_of(T_dev, B) == 0:
        return call_plan(B, Hkv, TS, device, num_warps, any_length=True)
    return plan_splits(B, Hkv, TS, device)


def append_token(x, c, T_dev):
    """x [B, H, 128] bf16 (channels contiguous): the step's token for every
    sequence of CompressedKV `c`, appended at row T_dev (one length for the
    batch, or one per sequence)."""
    if x.dtype != torch.bfloat16 or x.stride(-1) != 1 or tuple(x.shape) != (c.B, c.H, D):
        raise ValueError("x must be bf16 [B, H, 128] with contiguous channels")
    dev = x.device
    stream = torch.cuda.current_stream(dev).cuda_stream
    rc = lib.exk_append_token(x.data_ptr(), x.stride(0), x.stride(1), c.sm.data_ptr(), c.code.data_ptr(),
                              c.base.data_ptr(), c.rowmask.data_ptr(), c.rowoff.data_ptr(), c.raw.data_ptr(), c.cap,
                              c.cnt.data_ptr(), c.B, c.H, c.TS, T_dev.data_ptr(), _stride_of(T_dev, c.B),
                              status_tensor(dev.index).data_ptr(), dev.index, stream)
    check(rc, "exk_append_token")


def copy_from_host(dst, src):
    """dst (a contiguous CUDA tensor) <- src (a contiguous pinned CPU tensor of
    the same byte size): a kernel on the current stream reads the pinned
    memory over PCIe (exk_copy_from_host), so the copy needs no hand-off
    between the copy engine and the step's kernels. Returns dst."""
    if not (dst.is_cuda and dst.is_contiguous() and src.is_contiguous() and not src.is_cuda and src.is_pinned()):
        raise ValueError("dst must be a contiguous CUDA tensor and src a contiguous pinned host tensor")
    n = dst.numel() * dst.element_size()
    if src.numel() * src.element_size() != n:
        raise ValueError("dst and src must hold the same number of bytes")
    dev = dst.device
    check(lib.exk_copy_from_host(dst.data_ptr(), src.data_ptr(), n, dev.index,
                                 torch.cuda.current_stream(dev).cuda_stream), "exk_copy_from_host")
    return dst


def advance_length(T_dev, n=1):
    dev = T_dev.device
    check(lib.exk_advance_length(T_dev.data_ptr(), n, dev.index, torch.cuda.current_stream(dev).cuda_stream),
          "exk_advance_length")


def attention_compressed_devlen(q, kc, vc, T_dev, T_add=1, out=None, num_warps=None, advance=0):
    """Decode attention over the first min(TS, T_dev + T_add) tokens of the caches
    (T_dev: one int32 length for the batch or one per sequence), with the split
    plan's number of splits for their capacity TS, each sequence cut into that many
    equal page runs of its current length (see exk_attention_compressed_devlen); advance != 0
    then adds it to the batch length on the device (the end of a step)."""
    ka, TS, Hkv = _cache_args(kc)
    va, _, _ = _cache_args(vc)
    _check_q(q, TS, TS)
    B, Hq, _ = q.shape
    dev = q.device.index
    stream = torch.cuda.current_stream(q.device).cuda_stream
    ns, sl = devlen_plan(B, Hkv, TS, T_dev, dev, num_warps)
    ws = _workspace(q.device, stream, B * Hq, ns, sl)
    out = torch.empty_like(q) if out is None else _check_out(out, q)
    rc = lib.exk_attention_compressed_devlen(q.data_ptr(), ctypes.byref(ka), ctypes.byref(va), B, TS, Hkv, Hq, TS,
                                             T_dev.data_ptr(), T_add, _stride_of(T_dev, B), advance,
                                             ctypes.byref(ws[3]), out.data_ptr(), _consumer_warps(num_warps),
                                             D ** -0.5 * LOG2E, status_tensor(dev).data_ptr(), dev, stream)
    check(rc, "exk_attention_compressed_devlen")
    return out


# ----------------------------------------------------------------------------- paged caches

def _paged_warps(Hkv):
    """Consumer warps for a paged call: the head group (one page per head per stage)."""
    if Hkv % 8 == 0:
        return 8
    if Hkv % 4 == 0:
        return 4
    raise ValueError("paged attention needs a KV head count that is a multiple of 4")


def _paged_check(q, block_table, seq_lens):
    B = q.shape[0]
    for t, name in ((block_table, "block_table"), (seq_lens, "seq_lens")):
        if t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous CUDA int32 tensor")
    if block_table.dim() != 2 or block_table.shape[0] != B or seq_lens.shape != (B,):
        raise ValueError("block_table must be [B, max_pages] and seq_lens [B]")
    return block_table.shape[1]


def attention_paged(q, kc, vc, block_table, seq_lens, out=None):
    """Decode attention over paged caches: kc, vc are CompressedKV objects (or
    their .buffers() dicts) used as page pools — their [B', TS'] buffers seen as
    B' * TS' / 16 pages — block_table int32 [B, max_pages] names each
    sequence's pages in the pool, seq_lens int32 [B] its tokens (both on the
    device). Same results as attention_compressed_devlen over the same pages
    laid out contiguously (exk_attention_compressed_paged)."""
    ka, TS, Hkv = _cache_args(kc)
    va, _, _ = _cache_args(vc)
    Bp = kc["shape"][0] if isinstance(kc, dict) else kc.B
    max_pages = _paged_check(q, block_table, seq_lens)
    _check_q(q, max_pages * P, max_pages * P)
    B, Hq, _ = q.shape
    dev = q.device.index
    stream = torch.cuda.current_stream(q.device).cuda_stream
    ns, sl = plan_splits(B, Hkv, max_pages * P, dev)
    ws = _workspace(q.device, stream, B * Hq, ns, sl)
    out = torch.empty_like(q) if out is None else _check_out(out, q)
    rc = lib.exk_attention_compressed_paged(q.data_ptr(), ctypes.byref(ka), ctypes.byref(va), Bp * TS // P, Hkv, B,
                                            Hq, block_table.data_ptr(), max_pages, seq_lens.data_ptr(),
                                            ctypes.byref(ws[3]), out.data_ptr(), _paged_warps(Hkv),
                                            D ** -0.5 * LOG2E, status_tensor(dev).data_ptr(), dev, stream)
    check(rc, "exk_attention_compressed_paged")
    return out


def attention_reference_paged(q, k, v, block_table, seq_lens, out=None):
    """The bf16 sibling of attention_paged over bf16 pools k, v of shape
    [B', TS', Hkv, 128] (contiguous; pages of 16 rows), bit-identical for the
    same values."""
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16 or not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("k and v must be contiguous bf16 [B', TS', Hkv, 128]")
    Hkv = k.shape[-2]
    pool_pages = k.numel() // (Hkv * D * P)
    max_pages = _paged_check(q, block_table, seq_lens)
    _check_q(q, max_pages * P, max_pages * P)
    B, Hq, _ = q.shape
    dev = q.device.index
    stream = torch.cuda.current_stream(q.device).cuda_stream
    ns, sl = plan_splits(B, Hkv, max_pages * P, dev)
    ws = _workspace(q.device, stream, B * Hq, ns, sl)
    out = torch.empty_like(q) if out is None else _check_out(out, q)
    rc = lib.exk_attention_bf16_paged(q.data_ptr(), k.data_ptr(), v.data_ptr(), pool_pages, Hkv, B, Hq,
                                      block_table.data_ptr(), max_pages, seq_lens.data_ptr(), ctypes.byref(ws[3]),
                                      out.data_ptr(), _paged_warps(Hkv), D ** -0.5 * LOG2E,
                                      status_tensor(dev).data_ptr(), dev, stream)
    check(rc, "exk_attention_bf16_paged")
    return out


def attention_reference_devlen(q, k, v, T_dev, T_add=0, out=None, num_warps=None):
    """The bf16 sibling of attention_compressed_devlen on k, v [B, TS, Hkv, 128]
    (bit-identical for the same values, lengths and num_warps)."""
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16 or not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("k and v must be contiguous bf16 [B, TS, Hkv, 128]")
    TS, Hkv = k.shape[1], k.shape[2]
    _check_q(q, TS, TS)
    B, Hq, _ = q.shape
    dev = q.device.index
    stream = torch.cuda.current_stream(q.device).cuda_stream
    ns, sl = devlen_plan(B, Hkv, TS, T_dev, dev, num_warps)
    ws = _workspace(q.device, stream, B * Hq, ns, sl)
    out = torch.empty_like(q) if out is None else _check_out(out, q)
    rc = lib.exk_attention_bf16_devlen(q.data_ptr(), k.data_ptr(), v.data_ptr(), B, TS, Hkv, Hq, TS, T_dev.data_ptr(),
                                       T_add, _stride_of(T_dev, B), 0, ctypes.byref(ws[3]), out.data_ptr(),
                                       _consumer_warps(num_warps), D ** -0.5 * LOG2E,
                                       status_tensor(dev).data_ptr(), dev, stream)
    check(rc, "exk_attention_bf16_devlen")
    return out


# ----------------------------------------------------------------------------- new tokens into paged caches
#
# The paged calls below share one set of device tensors per step: block_table
# int32 [B, max_pages], seq_lens int32 [B] (each sequence's tokens, the new
# ones included) and, where sequences bring different numbers of new tokens,
# cu_seqlens int32 [B + 1] (sequence b's are rows cu_seqlens[b] ..
# cu_seqlens[b + 1] of the packed q, k, v). Rows past cu_seqlens[B] are left
# alone, so a captured step can serve a padded batch.

def rope_table(inv_freq, positions, scale=1.0):
    """cos_sin fp32 [positions, 128] of rope_append_paged for the 64 inverse
    frequencies inv_freq (a model's rotary_emb.inv_freq; its attention_scaling
    as `scale`): row p holds the cosines, then the sines, of p * inv_freq. The
    angles are formed in 64 bits."""
    if inv_freq.shape != (D // 2,):
        raise ValueError("inv_freq must hold 64 inverse frequencies")
    ang = torch.arange(positions, dtype=torch.float64, device=inv_freq.device)[:, None] * inv_freq.double()
    return (torch.cat([ang.cos(), ang.sin()], 1) * scale).float()


def _stream(dev):
    """The current stream of CUDA device number `dev` (torch.cuda.current_stream
    builds an object for it, a tenth of a small call's time)."""
    return torch._C._cuda_getCurrentRawStream(dev)


def _rows(t, name, n, heads, dev):
    """(address, token stride, head stride) of strided token rows [n, heads, 128] of a
    packed batch on CUDA device `dev`, checked."""
    shape, at = t.shape, t.data_ptr()
    if len(shape) != 3 or shape[0] != n or shape[1] != heads or shape[2] != D or t.dtype is not torch.bfloat16 or \
            t.device != dev or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA bf16 tensor [{n}, {heads}, {D}] on {dev}")
    st, sh, sc = t.stride()
    if sc != 1 or st % 8 or sh % 8 or at % 16 or st < 0 or sh <= 0 or (st == 0 and n > 1):
        raise ValueError(f"{name}: channels must be contiguous, token and head strides positive multiples of 8 elements "
                         "and rows 16-byte aligned")
    return at, st or heads * D, sh


def _index(t, name, shape, dev):
    """Address of a contiguous int32 tensor of `shape` on `dev`, checked."""
    if t.dtype is not torch.int32 or t.device != dev or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor {list(shape)} on {dev}")
    return t.data_ptr()


def _heads(q, Hkv):
    """(tokens, query heads) of packed queries, a multiple of Hkv."""
    if q.dim() != 3 or q.shape[1] % Hkv:
        raise ValueError(f"q must be [N, Hq, {D}] with Hq a multiple of the {Hkv} KV heads")
    return q.shape[0], q.shape[1]


def _new_rows(out, name, q, N, Hq):
    """The output for q's rows: `out`, checked, or a new tensor, with its address and strides."""
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        return out, (out.data_ptr(), Hq * D, D)
    return out, _rows(out, name, N, Hq, q.device)


def _append_args(q, k, v, cos_sin, block_table, seq_lens, cu_seqlens, slots, q_norm, k_norm, eps, q_out, Hkv, pool_pages):
    """exk_append of a call, checked; its output; tokens and sequences."""
    dev = q.device
    N, Hq = _heads(q, Hkv)
    q_at, q_st, q_sh = _rows(q, "q", N, Hq, dev)
    k_at, k_st, k_sh = _rows(k, "k", N, Hkv, dev)
    v_at, v_st, v_sh = _rows(v, "v", N, Hkv, dev)
    if block_table.dim() != 2:
        raise ValueError("block_table must be [B, max_pages]")
    B, max_pages = block_table.shape
    if cu_seqlens is None and B != N:
        raise ValueError("without cu_seqlens every sequence brings one token: q must be [B, heads, 128]")
    if cos_sin.dim() != 2 or cos_sin.shape[1] != D or cos_sin.dtype is not torch.float32 or cos_sin.device != dev or \
            not cos_sin.is_contiguous():
        raise ValueError(f"cos_sin must be a contiguous fp32 tensor [positions, {D}] on {dev}")
    if (q_norm is None) != (k_norm is None):
        raise ValueError("q_norm and k_norm come together")
    wq = wk = 0
    if q_norm is not None:
        for w in (q_norm, k_norm):
            if w.dtype is not torch.bfloat16 or w.shape != (D,) or w.device != dev or not w.is_contiguous() or \
                    w.data_ptr() % 8:
                raise ValueError(f"q_norm and k_norm must be contiguous, 8-byte aligned bf16 tensors [{D}] on {dev}")
        wq, wk = q_norm.data_ptr(), k_norm.data_ptr()
    q_out, (o_at, o_st, o_sh) = _new_rows(q_out, "q_out", q, N, Hq)
    a = APPEND.pack(q_at, k_at, v_at, o_at, q_st, q_sh, k_st, k_sh, v_st, v_sh, o_st, o_sh, cos_sin.data_ptr(), wq, wk,
                    0 if cu_seqlens is None else _index(cu_seqlens, "cu_seqlens", (B + 1,), dev),
                    _index(seq_lens, "seq_lens", (B,), dev), _index(block_table, "block_table", (B, max_pages), dev),
                    0 if slots is None else _index(slots, "slots", (B,), dev),
                    N, B, Hq, Hkv, cos_sin.shape[0], max_pages, pool_pages, eps)
    return a, q_out, N, B


def _bf16_pool(k, v, q):
    """(KV heads, pages) of a pair of bf16 pools [B', TS', Hkv, 128]."""
    shape, dev = k.shape, q.device
    if len(shape) != 4 or shape[3] != D or v.shape != shape or k.dtype is not torch.bfloat16 or \
            v.dtype is not torch.bfloat16 or k.device != dev or v.device != dev or \
            not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("k and v pools must be contiguous bf16 [B', TS', Hkv, 128] on q's device")
    B, TS, H, _ = shape
    if TS % P or B * TS * H == 0:
        raise ValueError("a pool's TS' must be a positive multiple of 16")
    return H, B * TS // P


def _coded_pool(c, dev, write):
    """(exk_cview, KV heads, pages, slots of the raw pool, counter) of a cache used as a
    page pool: a cache object, or a dict of its buffers."""
    if isinstance(c, dict):
        sm, raw, cap, cnt = c["sm"], c["raw"], c.get("cap"), c.get("cnt")
        B, TS, H = c["shape"][:3]
        view = CVIEW.pack(sm.data_ptr(), c["code"].data_ptr(), c["base"].data_ptr(), c["rowmask"].data_ptr(),
                          c["rowoff"].data_ptr(), raw.data_ptr(), raw.shape[0])
    else:
        view, TS, H = _cache_args(c)
        view = ctypes.byref(view)
        B, sm, cap, cnt = c.B, c.sm, getattr(c, "cap", None), getattr(c, "cnt", None)
    if sm.device != dev:
        raise ValueError("the pools must be on q's device")
    if write and (cap is None or cnt is None or cnt.dtype is not torch.int32 or cnt.device != dev):
        raise ValueError("a pool that is written needs its raw pool's capacity (cap) and int32 counter (cnt)")
    return view, H, B * TS // P, cap, cnt


def rope_append_paged(q, k, v, cos_sin, kc, vc, block_table, seq_lens, cu_seqlens=None, slots=None, q_norm=None,
                      k_norm=None, eps=1e-6, q_out=None):
    """Rotates a batch's new queries and keys at their positions and stores keys
    and values in their sequences' pages of the compressed pools kc, vc (a
    PagedCompressedKV, any CompressedKV seen as pages, or a dict of their
    buffers with cap and cnt). q [N, Hq, 128], k, v [N, Hkv, 128] bf16, packed
    by cu_seqlens (None: one token per sequence); channels contiguous, other
    strides free (views of a fused projection). Sequence b's new tokens are its
    last: positions seq_lens[b] - n_b .. seq_lens[b] - 1. cos_sin: rope_table().
    q_norm, k_norm (bf16 [128], both or neither): RMS norm per head first.
    Pages that fill are encoded; each sequence's last, unfilled page stays raw
    in tail slot slots[b] (default b), where the next call looks for it (after a
    sequence was cut back: cut_back_paged() first). The caller keeps (N + 15 * B) * Hkv
    raw rows free (PagedCompressedKV.ensure_headroom(N)); where they run out, cnt
    exceeds cap and readers report the pages that had no room. Returns the rotated
    queries [N, Hq, 128] (q_out, which may be q). Positions or pages out of
    range are not stored and reported by check_status()."""
    kv, H, pages, k_cap, k_cnt = _coded_pool(kc, q.device, True)
    vv, vH, v_pages, v_cap, v_cnt = _coded_pool(vc, q.device, True)
    if vH != H or v_pages != pages:
        raise ValueError("the key and value pools differ in shape")
    a, q_out, N, B = _append_args(q, k, v, cos_sin, block_table, seq_lens, cu_seqlens, slots, q_norm, k_norm, eps, q_out,
                                  H, pages)
    if N == 0:
        return q_out
    n = lib.exk_rope_append_scratch(N, B, H, cu_seqlens is not None)
    scratch = torch.empty(n, dtype=torch.uint8, device=q.device)
    dev = q.device.index
    check(lib.exk_rope_append_compressed(a, kv, k_cap, k_cnt.data_ptr(), vv,
                                         v_cap, v_cnt.data_ptr(), scratch.data_ptr(), n,
                                         status_tensor(dev).data_ptr(), dev,
                                         _stream(dev)), "exk_rope_append_compressed")
    return q_out


def cut_back_paged(kc, vc, block_table, seq_lens, slots=None):
    """After sequences of the compressed pools kc, vc were cut back to seq_lens [B]
    tokens (drafts that were not taken) and before the next rope_append_paged: a
    page that had been completed and now ends the sequence is opened again, its
    rows in tail slot slots[b] (default b). Sequences whose last page is open, or
    whole, are left alone, so every sequence of a step may go through it; one
    launch, no sync. (bf16 pools need nothing of the kind.)"""
    dev = block_table.device
    kv, H, pages, k_cap, _ = _coded_pool(kc, dev, True)
    vv, vH, v_pages, v_cap, _ = _coded_pool(vc, dev, True)
    if vH != H or v_pages != pages:
        raise ValueError("the key and value pools differ in shape")
    if block_table.dim() != 2 or block_table.shape[1] == 0 or not block_table.is_cuda:
        raise ValueError("block_table must be a CUDA tensor [B, max_pages]")
    B, max_pages = block_table.shape
    table = _index(block_table, "block_table", (B, max_pages), dev)
    lens = _index(seq_lens, "seq_lens", (B,), dev)
    at = 0 if slots is None else _index(slots, "slots", (B,), dev)
    if B == 0:
        return
    check(lib.exk_reopen_pages(table, B, max_pages, pages, H, lens, at, kv, k_cap, vv, v_cap,
                               status_tensor(dev.index).data_ptr(), dev.index, _stream(dev.index)), "exk_reopen_pages")


def rope_append_reference_paged(q, k, v, cos_sin, k_pool, v_pool, block_table, seq_lens, cu_seqlens=None, q_norm=None,
                                k_norm=None, eps=1e-6, q_out=None):
    """The bf16 sibling of rope_append_paged over bf16 pools [B', TS', Hkv, 128]
    (pages of 16 rows): the same values in the same places."""
    H, pages = _bf16_pool(k_pool, v_pool, q)
    a, q_out, N, _ = _append_args(q, k, v, cos_sin, block_table, seq_lens, cu_seqlens, None, q_norm, k_norm, eps, q_out,
                                  H, pages)
    if N == 0:
        return q_out
    dev = q.device.index
    check(lib.exk_rope_append_bf16(a, k_pool.data_ptr(), v_pool.data_ptr(), status_tensor(dev).data_ptr(),
                                   dev, _stream(dev)), "exk_rope_append_bf16")
    return q_out


# ----------------------------------------------------------------------------- prompt attention

def _prefill_args(q, cu_seqlens, Hkv, max_keys, out):
    """exk_prefill of a call, checked; its output; tokens and sequences; and the
    workspace it names, which belongs to the call (inside a capture: to the
    graph), so no two calls share it."""
    dev = q.device
    N, Hq = _heads(q, Hkv)
    q_at, q_st, q_sh = _rows(q, "q", N, Hq, dev)
    B = cu_seqlens.numel() - 1
    if B < 1:
        raise ValueError("cu_seqlens must hold B + 1 offsets")
    cu = _index(cu_seqlens, "cu_seqlens", (B + 1,), dev)
    out, (o_at, o_st, o_sh) = _new_rows(out, "out", q, N, Hq)
    ns = 1
    if max_keys > 896:                      # (a split has at least four tiles of 128 keys)
        ns = lib.exk_prefill_splits(N, B, Hq, Hkv, max_keys, num_sms(dev.index))
        if ns < 0:
            check(ns, "exk_prefill_splits")
    ws, o, m, l = None, 0, 0, 0
    if ns > 1:
        rows = N * Hq * ns
        ws = torch.empty(rows * (D + 2), dtype=torch.float32, device=dev)
        o = ws.data_ptr()
        m, l = o + rows * D * 4, o + rows * (D + 1) * 4
    a = PREFILL.pack(q_at, o_at, q_st, q_sh, o_st, o_sh, cu, o, m, l, N, B, Hq, Hkv, ns, D ** -0.5 * LOG2E)
    return a, out, N, B, ws


def attention_prefill(q, k, v, cu_seqlens, cu_seqlens_k=None, out=None):
    """Causal attention of packed prompts: q [N, Hq, 128], k, v [Nk, Hkv, 128] bf16
    (channels contiguous, other strides free), sequence b's rows
    cu_seqlens[b] .. cu_seqlens[b + 1] (int32 [B + 1], device) of q and
    cu_seqlens_k[b] .. (default cu_seqlens) of k and v. A sequence's last query
    sees its last key, so with more keys than queries each query sees the
    excess as context; a query that sees no key gives zeros. Up to 16 query
    heads per KV head. Returns bf16 [N, Hq, 128] (`out`, which may be q); rows
    past cu_seqlens[B] are left as they were."""
    if k.dim() != 3 or k.shape[0] == 0 or k.shape[1] == 0:
        raise ValueError("k and v must be [Nk, Hkv, 128] with at least one row")
    Nk, Hkv = k.shape[:2]
    k_at, k_st, k_sh = _rows(k, "k", Nk, Hkv, q.device)
    v_at, v_st, v_sh = _rows(v, "v", Nk, Hkv, q.device)
    # (the plan only: the lengths are on the device, a sequence has Nk / B keys in the mean)
    a, out, N, B, ws = _prefill_args(q, cu_seqlens, Hkv, -(-Nk // max(1, cu_seqlens.numel() - 1)), out)
    if cu_seqlens_k is None:
        if Nk != N:
            raise ValueError("k and v rows differ from q's: give cu_seqlens_k")
        cu_k = cu_seqlens.data_ptr()
    else:
        cu_k = _index(cu_seqlens_k, "cu_seqlens_k", (B + 1,), q.device)
    if N == 0:
        return out
    dev = q.device.index
    check(lib.exk_attention_prefill(a, k_at, k_st, k_sh, v_at, v_st, v_sh, Nk, cu_k,
                                    status_tensor(dev).data_ptr(), dev,
                                    _stream(dev)), "exk_attention_prefill")
    return out


def _most_keys(block_table, max_len):
    """Keys a sequence of the call may have: max_len rounded up to whole pages, or all its pages."""
    if block_table.dim() != 2 or block_table.shape[1] == 0:
        raise ValueError("block_table must be [B, max_pages]")
    cap = block_table.shape[1] * P
    rows = cap if max_len is None else -(-max_len // P) * P
    if not 0 < rows <= cap:
        raise ValueError(f"max_len={max_len} out of range (1..{cap})")
    return rows


def _check_pages(block_table, seq_lens, B, dev):
    max_pages = block_table.shape[1]
    return (_index(block_table, "block_table", (B, max_pages), dev), max_pages,
            _index(seq_lens, "seq_lens", (B,), dev))


def attention_prefill_paged(q, kc, vc, block_table, seq_lens, cu_seqlens, max_len=None, out=None):
    """attention_prefill with the keys and values in compressed pools (as
    attention_paged takes them): the queries are the last tokens of sequences of
    seq_lens[b] tokens whose pages block_table names, as rope_append_paged left
    them. max_len (host, at least every seq_lens[b]; default max_pages * 16)
    bounds the workspace of B * max_len decoded rows; a longer sequence is cut
    and reported by check_status(). Sequences without queries in the call are
    not read, whatever their lengths and pages. Bit-identical to
    attention_prefill_reference_paged for the same values and max_len."""
    kv, H, pages, _, _ = _coded_pool(kc, q.device, False)
    vv, vH, v_pages, _, _ = _coded_pool(vc, q.device, False)
    if vH != H or v_pages != pages:
        raise ValueError("the key and value pools differ in shape")
    rows = _most_keys(block_table, max_len)
    a, out, N, B, ws = _prefill_args(q, cu_seqlens, H, rows, out)
    table, max_pages, lens = _check_pages(block_table, seq_lens, B, q.device)
    if N == 0:
        return out
    kv_rows = torch.empty(2, B * rows, H, D, dtype=torch.bfloat16, device=q.device)
    dev = q.device.index
    check(lib.exk_attention_prefill_paged_compressed(
        a, kv, vv, pages, table, max_pages, lens, kv_rows[0].data_ptr(),
        kv_rows[1].data_ptr(), rows, status_tensor(dev).data_ptr(), dev,
        _stream(dev)), "exk_attention_prefill_paged_compressed")
    return out


def attention_prefill_reference_paged(q, k, v, block_table, seq_lens, cu_seqlens, max_len=None, out=None):
    """The bf16 sibling of attention_prefill_paged over bf16 pools k, v [B', TS',
    Hkv, 128] (pages of 16 rows), read in place: no workspace of rows, and max_len
    only bounds the plan of the splits."""
    H, pages = _bf16_pool(k, v, q)
    a, out, N, B, ws = _prefill_args(q, cu_seqlens, H, _most_keys(block_table, max_len), out)
    table, max_pages, lens = _check_pages(block_table, seq_lens, B, q.device)
    if N == 0:
        return out
    dev = q.device.index
    check(lib.exk_attention_prefill_paged(a, k.data_ptr(), v.data_ptr(), pages, table, max_pages, lens,
                                          status_tensor(dev).data_ptr(), dev,
                                          _stream(dev)),
          "exk_attention_prefill_paged")
    return out
