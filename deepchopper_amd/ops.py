"""Tensor-level wrappers over the C ABI.

torch is used here only as plumbing: device allocations, the current HIP stream and host<->device
copies.  All arithmetic happens inside libdeepchopper_hip.so.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import os

import numpy as np
import torch

from . import _lib

SM_MAX_LEN = 65536  # longest read the smoothing kernel's LDS bit-vectors hold (csrc/smooth.hip)


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: torch.Tensor | None) -> int | None:
    if t is None:
        return None
    assert t.is_cuda and t.is_contiguous(), "device-resident contiguous tensor required"
    return t.data_ptr()


def _dev() -> torch.device:
    _lib.require_gpu()
    return torch.device("cuda", torch.cuda.current_device())


def pack_reads(reads: list[bytes]) -> tuple[np.ndarray, np.ndarray]:
    """Concatenate byte strings -> (uint8 buffer, int64 offsets[n+1])."""
    lens = np.fromiter((len(r) for r in reads), dtype=np.int64, count=len(reads))
    offs = np.zeros(len(reads) + 1, dtype=np.int64)
    np.cumsum(lens, out=offs[1:])
    buf = np.frombuffer(b"".join(reads), dtype=np.uint8) if len(reads) else np.zeros(0, np.uint8)
    return buf, offs


def to_device(a: np.ndarray) -> torch.Tensor:
    a = np.ascontiguousarray(a)
    if not a.flags.writeable:
        a = a.copy()
    t = torch.from_numpy(a)
    return t.to(_dev(), non_blocking=False)


def pt_pack(logits, labels, input_ids, input_quals, table: np.ndarray, out: torch.Tensor) -> None:
    """dc_pt_pack on the current stream: the storages data/0..3 of every `.pt` file of a fused launch, cut out of the launch's
    dense device arrays and laid out as the files hold them, at the files' offsets of `out` (uint8, device).
    `table`: int64 [n_files, 4] = row0, rows, first column, byte offset (multiple of 64) -- host array; uploaded here."""
    table = np.ascontiguousarray(table, np.int64)
    d_table = torch.from_numpy(table).pin_memory().to(logits.device, non_blocking=True)  # (no wait for the stream's earlier work)
    n, stride = input_ids.shape
    assert logits.is_contiguous() and labels.is_contiguous() and input_ids.is_contiguous() and input_quals.is_contiguous()
    assert logits.shape == (n, stride, 2) and labels.dtype == torch.int8 and out.dtype == torch.uint8 and out.is_contiguous()
    _lib.check(_lib.lib().dc_pt_pack(_stream(), _ptr(logits), _ptr(labels), _ptr(input_ids), int(input_ids.dtype == torch.int64),
                                     _ptr(input_quals), n, stride, int(table.shape[0]), C.c_void_p(table.ctypes.data), _ptr(d_table),
                                     _ptr(out), out.numel()))


# ------------------------------------------------------------------------------------------
# tokenise
# ------------------------------------------------------------------------------------------
def normalize_seq_batch(seq: torch.Tensor, offsets: torch.Tensor, iupac: bool):
    n = offsets.numel() - 1
    out = torch.empty_like(seq)
    out_len = torch.empty(n, dtype=torch.int32, device=seq.device)
    _lib.check(_lib.lib().dc_normalize_seq(_stream(), _ptr(seq), _ptr(offsets), n, int(iupac), _ptr(out), _ptr(out_len)))
    return out, out_len


def encode_qual_bytes(qual: torch.Tensor, qual_offset: int) -> torch.Tensor:
    out = torch.empty_like(qual)
    _lib.check(_lib.lib().dc_encode_qual(_stream(), _ptr(qual), qual.numel(), qual_offset, _ptr(out)))
    return out


def tokenize_batch(seq, qual, offsets, *, max_length: int, row_stride: int, pad_left: bool = True,
                   ids_i64: bool = True, qual_offset: int = 33, want_labels: bool = True):
    """Fused T1-T5.  Returns dict(input_ids, input_quals, labels, n_tokens, status)."""
    n = offsets.numel() - 1
    dev = seq.device
    ids = torch.empty((n, row_stride), dtype=torch.int64 if ids_i64 else torch.uint8, device=dev)
    quals = torch.empty((n, row_stride), dtype=torch.float32, device=dev)
    labels = torch.empty((n, row_stride), dtype=torch.int8, device=dev) if want_labels else None
    ntok = torch.empty(n, dtype=torch.int32, device=dev)
    status = torch.empty(n, dtype=torch.int32, device=dev)
    _lib.check(_lib.lib().dc_tokenize_batch(
        _stream(), _ptr(seq), _ptr(qual), _ptr(offsets), n, max_length, qual_offset, row_stride,
        int(pad_left), int(ids_i64), _ptr(ids), _ptr(quals), _ptr(labels), _ptr(ntok), _ptr(status)))
    return {"input_ids": ids, "input_quals": quals, "labels": labels, "n_tokens": ntok, "status": status}


# ------------------------------------------------------------------------------------------
# k-mer encoder
# ------------------------------------------------------------------------------------------
def kmer_validate(seq, offsets, k: int, bases: bytes) -> torch.Tensor:
    n = offsets.numel() - 1
    status = torch.empty(n, dtype=torch.int32, device=seq.device)
    _lib.check(_lib.lib().dc_kmer_validate(_stream(), _ptr(seq), _ptr(offsets), n, k, bases, len(bases), _ptr(status)))
    return status


def kmer_encode(seq, qual, offsets, out_row, n_rows: int, k: int, bases: bytes, qual_offset: int, width: int,
                max_seq_len: int):
    n = offsets.numel() - 1
    dev = seq.device
    inp = torch.empty((n_rows, 2, width), dtype=torch.int32, device=dev)
    qout = torch.empty((n_rows, max_seq_len), dtype=torch.int32, device=dev)
    _lib.check(_lib.lib().dc_kmer_encode(_stream(), _ptr(seq), _ptr(qual), _ptr(offsets), _ptr(out_row), n, k, bases,
                                         len(bases), qual_offset, width, max_seq_len, _ptr(inp), _ptr(qout)))
    return inp, qout


def kmer_vectorize_targets(ranges: torch.Tensor, width: int) -> torch.Tensor:
    n_rows, n_targets, _ = ranges.shape
    out = torch.empty((n_rows, n_targets, width), dtype=torch.int32, device=ranges.device)
    _lib.check(_lib.lib().dc_kmer_vectorize_targets(_stream(), _ptr(ranges), n_rows, n_targets, width, _ptr(out)))
    return out


# ------------------------------------------------------------------------------------------
# smoothing / intervals
# ------------------------------------------------------------------------------------------
def smooth_intervals_from_logits(logits, first, length, *, window=21, min_interval=13, approved=20,
                                 max_intervals=None, want_labels=True, out_offsets=None, total: int | None = None):
    """logits f32[n_rows, row_stride, 2]; first/length int32[n].  Returns dict with pred / smooth
    (ragged int8 at out_offsets), intervals [n, max_intervals, 2], n_intervals, keep, n_keep."""
    n = first.numel()
    dev = logits.device
    max_intervals = max_intervals or max(approved, 1)
    row_stride = logits.shape[1]
    if want_labels and out_offsets is None:
        out_offsets = torch.zeros(n + 1, dtype=torch.int64, device=dev)
        out_offsets[1:] = torch.cumsum(length.to(torch.int64), 0)
    if not want_labels:
        total = 0
    elif total is None:  # callers that know the host-side sum pass it: reading it back would block on the forward
        total = int(out_offsets[-1].item())
    pred = torch.empty(total, dtype=torch.int8, device=dev) if want_labels else None
    smooth = torch.empty(total, dtype=torch.int8, device=dev) if want_labels else None
    iv = torch.zeros((n, max_intervals, 2), dtype=torch.int32, device=dev)
    niv = torch.empty(n, dtype=torch.int32, device=dev)
    keep = torch.zeros((n, max_intervals + 1, 2), dtype=torch.int32, device=dev)
    nkeep = torch.empty(n, dtype=torch.int32, device=dev)
    _lib.check(_lib.lib().dc_smooth_intervals_from_logits(
        _stream(), _ptr(logits), row_stride, _ptr(first), _ptr(length), n, _ptr(out_offsets), window, min_interval,
        approved, max_intervals, _ptr(pred), _ptr(smooth), _ptr(iv), _ptr(niv), _ptr(keep), _ptr(nkeep)))
    return {"pred": pred, "smooth": smooth, "offsets": out_offsets, "intervals": iv, "n_intervals": niv,
            "keep": keep, "n_keep": nkeep}


def smooth_intervals_from_labels(labels, offsets, *, window=21, min_interval=13, approved=20,
                                 apply_approved_rule=True, max_intervals=None, want_smooth=True):
    n = offsets.numel() - 1
    dev = labels.device
    max_intervals = max_intervals or max(approved, 1)
    smooth = torch.empty_like(labels) if want_smooth else None
    iv = torch.zeros((n, max_intervals, 2), dtype=torch.int32, device=dev)
    niv = torch.empty(n, dtype=torch.int32, device=dev)
    keep = torch.zeros((n, max_intervals + 1, 2), dtype=torch.int32, device=dev)
    nkeep = torch.empty(n, dtype=torch.int32, device=dev)
    _lib.check(_lib.lib().dc_smooth_intervals_from_labels(
        _stream(), _ptr(labels), _ptr(offsets), n, window, min_interval, approved, int(apply_approved_rule),
        max_intervals, _ptr(smooth), _ptr(iv), _ptr(niv), _ptr(keep), _ptr(nkeep)))
    return {"smooth": smooth, "intervals": iv, "n_intervals": niv, "keep": keep, "n_keep": nkeep}


def summary_predict_dense(pred: torch.Tensor, labels: torch.Tensor, ignore_label: int = -100):
    """pred/labels int8[n_rows, row_stride] -> (compacted pred, compacted labels, offsets)."""
    n_rows, row_stride = pred.shape
    dev = pred.device
    counts = torch.empty(n_rows, dtype=torch.int32, device=dev)
    L = _lib.lib()
    _lib.check(L.dc_summary_predict(_stream(), _ptr(pred), _ptr(labels), n_rows, row_stride, ignore_label, None, None,
                                    None, _ptr(counts)))
    offs = torch.zeros(n_rows + 1, dtype=torch.int64, device=dev)
    offs[1:] = torch.cumsum(counts.to(torch.int64), 0)
    total = int(offs[-1].item())
    op = torch.empty(total, dtype=torch.int8, device=dev)
    ol = torch.empty(total, dtype=torch.int8, device=dev)
    _lib.check(L.dc_summary_predict(_stream(), _ptr(pred), _ptr(labels), n_rows, row_stride, ignore_label, _ptr(offs),
                                    _ptr(op), _ptr(ol), _ptr(counts)))
    return op, ol, offs


# ------------------------------------------------------------------------------------------
# sequence-layer and scoring operators.  None of them is recorded by torch's autograd: the gradients are the *_backward functions', and a call
# whose inputs autograd would follow is refused.
# ------------------------------------------------------------------------------------------
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_TOKEN_TYPES = {torch.int8: 0, torch.uint8: 1, torch.int32: 2, torch.int64: 3}
_NORM_KINDS = {"layer": 0, "rms": 1}
_GATE_ACTS = {"identity": 0, "sigmoid": 1, "silu": 2}
STATS_FROM = 513  # DC_STATS_FROM: classes from which token_logprobs_backward needs the forward's statistics
_NO_SWITCH = contextlib.nullcontext()
try:  # (plain integers, a tenth of the cost of the objects torch.cuda makes of them: a step of a few tokens is as long as its call)
    from torch._C import _cuda_getCurrentRawStream as _stream_of, _cuda_getDevice as _current_device
except ImportError:
    def _stream_of(dev: int) -> int:
        return torch.cuda.current_stream(dev).cuda_stream

    _current_device = torch.cuda.current_device


def _device_of(name: str, t: torch.Tensor) -> int:
    if not t.is_cuda:
        raise ValueError(f"{name}: device-resident tensor required, got one on {t.device}")
    return t.get_device()


def _on(dev: int):
    """Context in which device `dev` is the current one (a call's kernels run on ITS tensors' device, on that device's current stream)."""
    return _NO_SWITCH if dev == _current_device() else torch.cuda.device(dev)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _not_recorded(name: str, *inputs: torch.Tensor | None) -> None:
    if torch.is_grad_enabled():
        for t in inputs:
            if t is not None and t.requires_grad:
                raise ValueError(f"{name}: an input requires gradients, but autograd does not record this operator: call it under torch.no_grad() or "
                                 f"with detached tensors, and take the gradients from {name}_backward")


def _like(dev: int, name: str, t: torch.Tensor | None, shape: tuple, dtype: torch.dtype) -> int | None:
    """Address of the contiguous tensor `t` (or None) after checking it against what the call needs."""
    if t is None:
        return None
    if t.get_device() != dev or t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous {dtype} tensor of shape {tuple(shape)} on cuda:{dev}, got {t.dtype} {tuple(t.shape)} "
                         f"with strides {t.stride()} on {t.device}")
    return t.data_ptr()


def _rows(dev: int, name: str, t: torch.Tensor | None, shape: torch.Size | None = None, dtype: torch.dtype | None = None) -> tuple[int | None, int]:
    """(address, elements between rows) of a [..., width] tensor whose rows are contiguous and evenly spaced (the halves of
    a projection, an expanded row), after checking it against the device, shape and type the call needs."""
    if t is None:
        return None, 0
    size = t.shape
    if t.get_device() != dev or (shape is not None and size != shape) or (t.dtype is not dtype if dtype is not None else t.dtype not in _DTYPES) or len(size) < 2:
        raise ValueError(f"{name}: expected {dtype or 'float32, float16 or bfloat16'} of shape {tuple(shape) if shape is not None else '[..., width]'} "
                         f"on cuda:{dev}, got {t.dtype} {tuple(size)} on {t.device}")
    if t.is_contiguous():
        return t.data_ptr(), size[-1]
    st = t.stride()
    if st[-1] != 1 and size[-1] > 1 and t.numel():
        raise ValueError(f"{name}: the last dimension must be contiguous (shape {tuple(size)}, strides {st})")
    # leading dimensions of size 1 say nothing about the distance of two rows
    dims = [(n, d) for n, d in zip(size[:-1], st[:-1]) if n != 1]
    for (_, outer), (n, d) in zip(dims, dims[1:]):
        if outer != n * d and t.numel():
            raise ValueError(f"{name}: rows must be evenly spaced (shape {tuple(size)}, strides {st})")
    return t.data_ptr(), dims[-1][1] if dims else size[-1]


def _apart(name: str, out: torch.Tensor, out_rows: tuple[int, int], other_name: str, other: torch.Tensor | None, rows: tuple[int | None, int],
           same: bool = False) -> None:
    """Refuses an output given by the caller that shares elements with an input: a kernel would read what another workgroup has written.
    `rows` as `_rows` returned them; `same`: the output may be that input itself, row for row."""
    if other is None or not out.numel() or out_rows[1] < out.shape[-1]:  # (rows that overlap among themselves are refused by the library)
        return
    width, n = out.shape[-1], out.numel() // out.shape[-1]
    ea, eb = out.element_size(), other.element_size()
    a, sa, b, sb = out_rows[0], out_rows[1] * ea, rows[0], rows[1] * eb
    wa, wb = width * ea, width * eb
    if a >= b + (n - 1) * sb + wb or b >= a + (n - 1) * sa + wa or (same and a == b and sa == sb and ea == eb):
        return
    if n > 1 and sa == sb and wa <= (b - a) % sa <= sa - wb:  # other columns of the same rows
        return
    starts, others = a + sa * np.arange(n), b + sb * np.arange(n)
    k = np.searchsorted(starts, others, side="right")  # rows k - 1 and k of the output lie on either side of an input's row's start
    if ((k > 0) & (starts[np.maximum(k, 1) - 1] + wa > others)).any() or ((k < n) & (starts[np.minimum(k, n - 1)] < others + wb)).any():
        raise ValueError(f"{name}: shares elements with {other_name}")


def _new_like(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """A dense tensor of `t`'s shape and device (`empty_like` takes half the time of `empty`)."""
    return torch.empty_like(t) if t.dtype is dtype and t.is_contiguous() else t.new_empty(t.shape, dtype=dtype)


def _address(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _tokens(dev: int, tokens: torch.Tensor | None, lead: torch.Size) -> tuple[int | None, int]:
    if tokens is None:
        return None, 0
    kind = _TOKEN_TYPES.get(tokens.dtype)
    if kind is None:
        raise ValueError(f"tokens: int8, uint8, int32 or int64 required, got {tokens.dtype}")
    return _like(dev, "tokens", tokens, lead, tokens.dtype), kind


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None = None, *, n_top: int = 0, ignore_index: int = -100,
                   want_entropy: bool = True, save: bool = False) -> dict:
    """Log probability of a given token per row of logits [..., n_classes], the row's entropy and its `n_top` likeliest
    classes (`dc_token_logprobs`).  `tokens` [...] int8 / uint8 / int32 / int64 or None; rows whose token is `ignore_index`
    (labels of padding) are not read and give 0, alternatives -1.  Returns dict(logprob f32 or None, entropy f32 or None,
    top_ids i32, top_logprob f32 [..., n_top] or None, stats: what `token_logprobs_backward` needs (with `save`; None below STATS_FROM
    classes))."""
    _not_recorded("token_logprobs", logits)
    dev = _device_of("logits", logits)
    ptr, stride = _rows(dev, "logits", logits)
    lead, n_classes, dtype = logits.shape[:-1], logits.shape[-1], logits.dtype
    n = logits.numel() // n_classes if n_classes else 0
    tok, kind = _tokens(dev, tokens, lead)
    logprob = None if tokens is None else logits.new_empty(lead, dtype=torch.float32)
    entropy = None
    if want_entropy:
        entropy = torch.empty_like(logprob) if logprob is not None else logits.new_empty(lead, dtype=torch.float32)
    stats = logits.new_empty((n, 3), dtype=torch.float32) if save and n_classes >= STATS_FROM else None
    ids = logits.new_empty((*lead, n_top), dtype=torch.int32) if n_top > 0 else None
    top = logits.new_empty((*lead, n_top), dtype=torch.float32) if n_top > 0 else None
    L = _lib.lib()
    nb = L.dc_token_logprobs_workspace(n, n_classes, n_top) if n_classes >= STATS_FROM else 0
    ws = logits.new_empty(nb, dtype=torch.uint8) if nb else None
    with _on(dev):
        _lib.check(L.dc_token_logprobs(_stream_of(dev), ptr, _DTYPES[dtype], n, n_classes, stride, tok, kind, ignore_index, n_top, _address(logprob),
                                       _address(entropy), _address(stats), _address(ids), _address(top), _address(ws), nb))
    return {"logprob": logprob, "entropy": entropy, "top_ids": ids, "top_logprob": top, "stats": stats}


def token_logprobs_backward(logits: torch.Tensor, tokens: torch.Tensor | None, stats: torch.Tensor | None, grad_logprob: torch.Tensor | None,
                            grad_entropy: torch.Tensor | None = None, *, ignore_index: int = -100) -> torch.Tensor:
    """Gradient of the logits for gradients of `token_logprobs`' logprob and entropy (either None: zero); `stats` as it
    returned them with `save=True`."""
    dev = _device_of("logits", logits)
    ptr, stride = _rows(dev, "logits", logits)
    lead, n_classes = logits.shape[:-1], logits.shape[-1]
    n = logits.numel() // n_classes if n_classes else 0
    tok, kind = _tokens(dev, tokens, lead)
    st = _like(dev, "stats", stats, (n, 3), torch.float32)
    gl = _like(dev, "grad_logprob", grad_logprob, lead, torch.float32)
    gh = _like(dev, "grad_entropy", grad_entropy, lead, torch.float32)
    out = _new_like(logits, logits.dtype)
    with _on(dev):
        _lib.check(_lib.lib().dc_token_logprobs_backward(_stream_of(dev), ptr, _DTYPES[logits.dtype], n, n_classes, stride, tok, kind, ignore_index, st,
                                                         gl, gh, out.data_ptr(), n_classes))
    return out


def _scan_shape(dev: int, x: torch.Tensor, offsets, begin, end, max_len):
    """(tokens, channels, sequences, longest, address of begin, of end) of a gated_scan call."""
    if offsets is None and begin is None and end is None:
        _need(x.dim() == 3, "x: [n_seqs, length, n_channels] required without offsets")
        _need(max_len is None or max_len == x.shape[1], "max_len of dense sequences is their length")
        return x.shape[0] * x.shape[1], x.shape[2], x.shape[0], x.shape[1], None, None
    _need((offsets is None) == (begin is not None) and (begin is None) == (end is None), "either offsets, or begin and end")
    if offsets is not None:
        _need(offsets.dim() == 1 and offsets.numel() >= 1, "offsets: int64[n_seqs + 1] required")
        n = offsets.numel() - 1
        b = _like(dev, "offsets", offsets, (n + 1,), torch.int64)
        e = b + 8
    else:
        n = begin.numel()
        b, e = _like(dev, "begin", begin, (n,), torch.int64), _like(dev, "end", end, (n,), torch.int64)
    if max_len is None:  # read back: callers that know the longest sequence pass it (and need to inside a graph capture)
        lens = offsets.diff() if offsets is not None else end - begin
        max_len = max(int(lens.max().item()), 0) if n else 0
    return x.numel() // max(x.shape[-1], 1), x.shape[-1], n, int(max_len), b, e


def gated_scan(x: torch.Tensor, f: torch.Tensor, *, offsets: torch.Tensor | None = None, begin: torch.Tensor | None = None,
               end: torch.Tensor | None = None, max_len: int | None = None, h0: torch.Tensor | None = None, reverse: bool = False,
               save: bool = False, out: torch.Tensor | None = None, h_last: torch.Tensor | None = None) -> dict:
    """h_t = sigmoid(f_t) h_(t-1) + (1 - sigmoid(f_t)) x_t along every sequence, per channel (`dc_gated_scan`): the recurrent
    counterpart of the long convolution, for reads of any length, with a state to carry on with.

    x, f [n_seqs, length, n_channels] dense, or [n_tokens, n_channels] with the sequences at `offsets` int64[n_seqs + 1], or at
    `begin` / `end` int64[n_seqs] (left-padded rows: first column and end of each); n_seqs * ceil(n_channels / 64) is below 2^20.
    `h0` f32[n_seqs, n_channels] state to start from; `reverse`: from the sequences' ends.  `h_last` may be given (`h0` itself: a state
    kept in place while bases stream in); `out` (apart from x and f) keeps what stands in tokens of no sequence, which are zero
    otherwise.  `max_len`: no sequence is longer (found on the host, with a wait, where it is not given).  A sequence that is, or that
    leaves the tokens, is refused: NaN in its row of h_last and, with `offsets`, in its rows of y; with `begin` / `end` or a given `out`
    those stay as tokens of no sequence.  Returns dict(y, h_last, saved: for `gated_scan_backward`, with `save`)."""
    _not_recorded("gated_scan", x, f, h0)
    dev = _device_of("x", x)
    xp, xs = _rows(dev, "x", x)
    shape, dtype, device = x.shape, x.dtype, x.device
    fp, fs = _rows(dev, "f", f, shape, dtype)
    n, c, seqs, longest, b, e = _scan_shape(dev, x, offsets, begin, end, max_len)
    h0p = _like(dev, "h0", h0, (seqs, c), torch.float32)
    zero_rest = out is None and offsets is not None  # (dense sequences cover every token)
    given = out is not None
    if not given:
        out = _new_like(x, dtype) if begin is None else torch.zeros(shape, dtype=dtype, device=device)
    yp, ys = _rows(dev, "out", out, shape, dtype)
    if given:
        _apart("out", out, (yp, ys), "x", x, (xp, xs))
        _apart("out", out, (yp, ys), "f", f, (fp, fs))
    given = h_last is not None
    if not given:
        h_last = torch.empty_like(h0) if h0 is not None else x.new_empty((seqs, c), dtype=torch.float32)
    hp = _like(dev, "h_last", h_last, (seqs, c), torch.float32)
    if given and h0p is not None and h0p != hp:
        _apart("h_last", h_last, (hp, c), "h0", h0, (h0p, c))
    L = _lib.lib()
    saved = x.new_empty(L.dc_gated_scan_saved(n, c), dtype=torch.float32) if save else None
    nb = L.dc_gated_scan_workspace(n, c, seqs, longest) if longest > 1 else 0
    ws = x.new_empty(nb, dtype=torch.uint8) if nb else None
    with _on(dev):
        _lib.check(L.dc_gated_scan(_stream_of(dev), _DTYPES[dtype], xp, xs, fp, fs, n, c, b, e, seqs, longest, int(reverse), h0p, yp, ys, int(zero_rest),
                                   hp, _address(saved), _address(ws), nb))
    return {"y": out, "h_last": h_last, "saved": saved}


def gated_scan_backward(x: torch.Tensor, f: torch.Tensor, saved: torch.Tensor, grad_y: torch.Tensor, *, grad_h_last: torch.Tensor | None = None,
                        h0: torch.Tensor | None = None, offsets: torch.Tensor | None = None, begin: torch.Tensor | None = None,
                        end: torch.Tensor | None = None, max_len: int | None = None, reverse: bool = False) -> dict:
    """Gradients of `gated_scan` for `grad_y` (and `grad_h_last`): dict(grad_x, grad_f, grad_h0 f32[n_seqs, n_channels]).  The other
    arguments as in the forward call, `saved` as it returned it; tokens of no sequence get zeros, refused sequences what they get in y."""
    dev = _device_of("x", x)
    xp, xs = _rows(dev, "x", x)
    shape, dtype, device = x.shape, x.dtype, x.device
    fp, fs = _rows(dev, "f", f, shape, dtype)
    gp, gs = _rows(dev, "grad_y", grad_y, shape, dtype)
    n, c, seqs, longest, b, e = _scan_shape(dev, x, offsets, begin, end, max_len)
    L = _lib.lib()
    h0p = _like(dev, "h0", h0, (seqs, c), torch.float32)
    glp = _like(dev, "grad_h_last", grad_h_last, (seqs, c), torch.float32)
    sp = _like(dev, "saved", saved, (L.dc_gated_scan_saved(n, c),), torch.float32)
    if begin is None:
        gx, gf = _new_like(x, dtype), _new_like(f, dtype)
    else:
        gx, gf = torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device)
    gh = x.new_empty((seqs, c), dtype=torch.float32)
    nb = L.dc_gated_scan_workspace(n, c, seqs, longest)
    ws = x.new_empty(nb, dtype=torch.uint8) if nb else None
    with _on(dev):
        _lib.check(L.dc_gated_scan_backward(_stream_of(dev), _DTYPES[dtype], xp, xs, fp, fs, n, c, b, e, seqs, longest, int(reverse), h0p, sp, gp, gs,
                                            glp, gx.data_ptr(), c, gf.data_ptr(), c, int(offsets is not None), gh.data_ptr(), _address(ws), nb))
    return {"grad_x": gx, "grad_f": gf, "grad_h0": gh}


_NORM_VECTORS = ("grad_scale", "grad_post_weight", "grad_post_bias", "grad_pre_weight", "grad_pre_bias")


def _norm_ref(y, residual) -> torch.Tensor:
    ref = y if y is not None else residual
    _need(ref is not None, "block_norm: a block's output or a residual is required")
    return ref


def _norm_codes(kind: str, gate_act: str) -> tuple[int, int]:
    if kind not in _NORM_KINDS or gate_act not in _GATE_ACTS:
        raise ValueError(f"kind is one of {sorted(_NORM_KINDS)}, gate_act one of {sorted(_GATE_ACTS)}; got {kind!r}, {gate_act!r}")
    return _NORM_KINDS[kind], _GATE_ACTS[gate_act]


def block_norm(y: torch.Tensor | None, residual: torch.Tensor | None = None, gate: torch.Tensor | None = None, *, kind: str = "layer",
               gate_act: str = "sigmoid", scale: torch.Tensor | None = None, post: bool = True, post_weight: torch.Tensor | None = None,
               post_bias: torch.Tensor | None = None, pre: bool = True, pre_weight: torch.Tensor | None = None, pre_bias: torch.Tensor | None = None,
               eps: float = 1e-5, dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> dict:
    """What stands between two blocks, in one pass (`dc_block_norm`): r' = residual + scale * act(gate) * norm(y) and n = norm(r').

    y, gate [..., width] of one type, residual of that type or float32.  `post=False`: no norm behind the block; `pre=False`: none in
    front of the next (the last block); y None: the first norm of a model; residual None: r' is the block's output alone.  Norms are
    "layer" or "rms", gates "identity", "sigmoid" or "silu"; weights, biases and `scale` are float32[width].  `dtype`: of n where y is
    None (default: the residual's); `out`: where r' goes (an input of its type itself: in place).  Returns dict(residual: r', normed: n or None)."""
    _not_recorded("block_norm", y, residual, gate, scale, post_weight, post_bias, pre_weight, pre_bias)
    ref = _norm_ref(y, residual)
    dev = _device_of("residual" if y is None else "y", ref)
    k, act = _norm_codes(kind, gate_act)
    act_dtype = y.dtype if y is not None else dtype or ref.dtype
    res_dtype = residual.dtype if residual is not None else act_dtype
    _need(act_dtype in _DTYPES, "block_norm: float32, float16 or bfloat16 required")
    _need(gate is None or y is not None, "gate: without a block's output")
    shape = ref.shape
    w = shape[-1]
    yp, ys = _rows(dev, "y", y, shape)
    gp, gs = _rows(dev, "gate", gate, shape, act_dtype)
    rp, rs = _rows(dev, "residual", residual, shape)
    one = (w,)
    sc = _like(dev, "scale", scale, one, torch.float32)
    pw, pb = _like(dev, "post_weight", post_weight, one, torch.float32), _like(dev, "post_bias", post_bias, one, torch.float32)
    qw, qb = _like(dev, "pre_weight", pre_weight, one, torch.float32), _like(dev, "pre_bias", pre_bias, one, torch.float32)
    given = out is not None
    if out is None and y is not None:
        out = _new_like(residual if residual is not None else y, res_dtype)
    op, os_ = _rows(dev, "out", out, shape, res_dtype)
    if given:
        _apart("out", out, (op, os_), "y", y, (yp, ys), same=True)
        _apart("out", out, (op, os_), "gate", gate, (gp, gs), same=True)
        _apart("out", out, (op, os_), "residual", residual, (rp, rs), same=True)
    normed = _new_like(ref, act_dtype) if pre else None
    with _on(dev):
        _lib.check(_lib.lib().dc_block_norm(
            _stream_of(dev), _DTYPES[act_dtype], _DTYPES[res_dtype], ref.numel() // w if w else 0, w, k, eps, yp, ys, gp, gs, act, rp, rs, sc,
            int(post), pw, pb, qw, qb, op, os_, _address(normed), w))
    return {"residual": residual if out is None else out, "normed": normed}


def block_norm_backward(y: torch.Tensor | None, residual: torch.Tensor | None = None, gate: torch.Tensor | None = None, *,
                        grad_residual: torch.Tensor | None = None, grad_normed: torch.Tensor | None = None, kind: str = "layer",
                        gate_act: str = "sigmoid", scale: torch.Tensor | None = None, post: bool = True,
                        post_weight: torch.Tensor | None = None, post_bias: torch.Tensor | None = None, pre_weight: torch.Tensor | None = None,
                        pre_bias: torch.Tensor | None = None, eps: float = 1e-5) -> dict:
    """Gradients of `block_norm` for gradients of r' (`grad_residual`) and n (`grad_normed`), either None where it is not used.  The other
    arguments as in the forward call, `residual` as it was BEFORE it.  Returns dict(grad_y, grad_gate, grad_residual, and float32[width]
    grad_scale, grad_post_weight, grad_post_bias, grad_pre_weight, grad_pre_bias); None for what the call did not have."""
    ref = _norm_ref(y, residual)
    dev = _device_of("residual" if y is None else "y", ref)
    k, act = _norm_codes(kind, gate_act)
    act_dtype = y.dtype if y is not None else grad_normed.dtype if grad_normed is not None else ref.dtype
    res_dtype = residual.dtype if residual is not None else act_dtype
    _need(act_dtype in _DTYPES, "block_norm: float32, float16 or bfloat16 required")
    _need(gate is None or y is not None, "gate: without a block's output")
    shape = ref.shape
    w = shape[-1]
    n = ref.numel() // w if w else 0
    yp, ys = _rows(dev, "y", y, shape)
    gp, gs = _rows(dev, "gate", gate, shape, act_dtype)
    rp, rs = _rows(dev, "residual", residual, shape)
    grp, grs = _rows(dev, "grad_residual", grad_residual, shape, res_dtype)
    gnp, gns = _rows(dev, "grad_normed", grad_normed, shape, act_dtype)
    one = (w,)
    sc = _like(dev, "scale", scale, one, torch.float32)
    pw, pb = _like(dev, "post_weight", post_weight, one, torch.float32), _like(dev, "post_bias", post_bias, one, torch.float32)
    qw = _like(dev, "pre_weight", pre_weight, one, torch.float32)
    _like(dev, "pre_bias", pre_bias, one, torch.float32)

    normed = post and y is not None
    sums = ref.new_empty((5, w), dtype=torch.float32).unbind()
    wanted = (y is not None and scale is not None, normed and post_weight is not None, normed and post_bias is not None, pre_weight is not None,
              pre_bias is not None)
    vectors = [t if want else None for t, want in zip(sums, wanted)]
    gy = None if y is None else _new_like(y, act_dtype)
    gg = None if gate is None else _new_like(gate, act_dtype)
    gr = None if residual is None else _new_like(residual, res_dtype)
    L = _lib.lib()
    nb = L.dc_block_norm_workspace(n, w, _DTYPES[res_dtype])
    ws = ref.new_empty(nb, dtype=torch.uint8) if nb else None
    with _on(dev):
        _lib.check(L.dc_block_norm_backward(
            _stream_of(dev), _DTYPES[act_dtype], _DTYPES[res_dtype], n, w, k, eps, yp, ys, gp, gs, act, rp, rs, sc, int(post), pw, pb, qw, grp, grs,
            gnp, gns, _address(gy), _address(gg), _address(gr), *map(_address, vectors), _address(ws), nb))
    return {"grad_y": gy, "grad_gate": gg, "grad_residual": gr, **dict(zip(_NORM_VECTORS, vectors))}


# ------------------------------------------------------------------------------------------
# model handle
# ------------------------------------------------------------------------------------------
GEMM_MODES = ("f32", "bf16x6", "fp16x3")


class HipModel:
    """Owns a `dc_model*` (weights repacked on the device, filters, workspace)."""

    def __init__(self, state_dict: dict[str, np.ndarray], cfg):
        from .weights import BB, HD, required_keys

        _lib.require_gpu()
        missing = [k for k in required_keys(cfg) if k not in state_dict]
        if missing:
            raise KeyError(f"checkpoint is missing {len(missing)} tensors, e.g. {missing[:3]}")
        self.cfg = cfg
        keep = []  # keep numpy buffers alive during dc_model_create

        def fp(name, shape=None):
            a = np.ascontiguousarray(np.asarray(state_dict[name], dtype=np.float32))
            if shape is not None and tuple(a.reshape(-1).shape) != (int(np.prod(shape)),):
                raise ValueError(f"{name}: expected {shape}, got {a.shape}")
            keep.append(a)
            return a.ctypes.data_as(_lib.f32p)

        D, DI, H, fo, emb = cfg.d_model, cfg.d_inner, cfg.head_hidden, cfg.filter_order, cfg.emb_dim
        if cfg.num_inner_mlps != 2:
            raise ValueError("the HIP filter kernel is specialised for num_inner_mlps == 2")
        layers = (_lib.LayerWeights * cfg.n_layer)()
        for i in range(cfg.n_layer):
            p = BB + f"layers.{i}."
            m = p + "mixer."
            f = m + "filter_fn."
            lw = layers[i]
            lw.norm1_w, lw.norm1_b = fp(p + "norm1.weight", (D,)), fp(p + "norm1.bias", (D,))
            lw.norm2_w, lw.norm2_b = fp(p + "norm2.weight", (D,)), fp(p + "norm2.bias", (D,))
            lw.in_proj_w, lw.in_proj_b = fp(m + "in_proj.weight", (3 * D, D)), fp(m + "in_proj.bias", (3 * D,))
            lw.out_proj_w, lw.out_proj_b = fp(m + "out_proj.weight", (D, D)), fp(m + "out_proj.bias", (D,))
            lw.short_w, lw.short_b = fp(m + "short_filter.weight", (3 * D, 3)), fp(m + "short_filter.bias", (3 * D,))
            lw.filt_bias = fp(f + "bias", (D,))
            lw.pos_z, lw.pos_t = fp(f + "pos_emb.z", (cfg.max_seq_len, emb)), fp(f + "pos_emb.t", (cfg.max_seq_len,))
            lw.filt_w0, lw.filt_b0 = fp(f + "implicit_filter.0.weight", (fo, emb)), fp(f + "implicit_filter.0.bias", (fo,))
            lw.filt_w1, lw.filt_b1 = fp(f + "implicit_filter.2.weight", (fo, fo)), fp(f + "implicit_filter.2.bias", (fo,))
            lw.filt_w2, lw.filt_b2 = fp(f + "implicit_filter.4.weight", (fo, fo)), fp(f + "implicit_filter.4.bias", (fo,))
            lw.filt_w3 = fp(f + "implicit_filter.6.weight", (D, fo))
            lw.filt_freq0 = fp(f + "implicit_filter.1.freq", (fo,))
            lw.filt_freq1 = fp(f + "implicit_filter.3.freq", (fo,))
            lw.filt_freq2 = fp(f + "implicit_filter.5.freq", (fo,))
            lw.deltas = fp(f + "modulation.deltas", (D,))
            lw.fc1_w, lw.fc1_b = fp(p + "mlp.fc1.weight", (DI, D)), fp(p + "mlp.fc1.bias", (DI,))
            lw.fc2_w, lw.fc2_b = fp(p + "mlp.fc2.weight", (D, DI)), fp(p + "mlp.fc2.bias", (D,))
        w = _lib.ModelWeights()
        w.embedding = fp(BB + "embeddings.word_embeddings.weight", (cfg.padded_vocab, D))
        w.layers = layers
        w.ln_f_w, w.ln_f_b = fp(BB + "ln_f.weight", (D,)), fp(BB + "ln_f.bias", (D,))
        w.head_w1, w.head_b1 = fp(HD + "linear1.weight", (H, D)), fp(HD + "linear1.bias", (H,))
        w.head_w2, w.head_b2 = fp(HD + "linear2.weight", (H, H)), fp(HD + "linear2.bias", (H,))
        w.head_w3, w.head_b3 = fp(HD + "linear3.weight", (cfg.num_class, H)), fp(HD + "linear3.bias", (cfg.num_class,))
        c = _lib.ModelConfig(
            d_model=D, d_inner=DI, n_layer=cfg.n_layer, vocab=cfg.padded_vocab, filter_order=fo, emb_dim=emb,
            short_filter_order=cfg.short_filter_order, max_seq_len=cfg.max_seq_len, head_hidden=H,
            num_class=cfg.num_class, gelu_tanh=1 if cfg.gelu_approximate == "tanh" else 0,
            ln_eps=cfg.layer_norm_epsilon, filter_shift=cfg.filter_shift)
        handle = C.c_void_p()
        _lib.check(_lib.lib().dc_model_create(C.byref(c), C.byref(w), C.byref(handle)))
        self._h = handle
        mode = C.c_int32()
        _lib.check(_lib.lib().dc_model_get_gemm_mode(self._h, C.byref(mode)))  # $DC_GEMM_MODE is parsed by the library only
        self.gemm_mode = GEMM_MODES[mode.value]
        self.prefix_mode = "linear" if os.environ.get("DC_PREFIX_MODE") in ("linear", "2") else "exact"  # (the library reads the same variable)
        del keep

    def close(self):
        if getattr(self, "_h", None):
            _lib.lib().dc_model_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def forward(self, input_ids: torch.Tensor, input_quals: torch.Tensor, out: torch.Tensor | None = None):
        """Dense batch [B, L] -> logits f32[B, L, 2]."""
        assert input_ids.dim() == 2 and input_ids.shape == input_quals.shape
        assert input_ids.dtype in (torch.int64, torch.uint8) and input_quals.dtype == torch.float32
        B, L = input_ids.shape
        if out is None:
            out = torch.empty((B, L, self.cfg.num_class), dtype=torch.float32, device=input_ids.device)
        _lib.check(_lib.lib().dc_forward(self._h, _stream(), _ptr(input_ids), int(input_ids.dtype == torch.int64),
                                         _ptr(input_quals), B, L, _ptr(out)))
        return out

    def forward_ragged(self, input_ids, input_quals, first: np.ndarray, n_tokens: np.ndarray, out=None):
        """Only tokens [first[r], first[r]+n_tokens[r]) of each row go through the model."""
        n, row_stride = input_ids.shape
        first = np.ascontiguousarray(first, dtype=np.int32)
        n_tokens = np.ascontiguousarray(n_tokens, dtype=np.int32)
        if out is None:
            out = torch.zeros((n, row_stride, self.cfg.num_class), dtype=torch.float32, device=input_ids.device)
        _lib.check(_lib.lib().dc_forward_ragged(
            self._h, _stream(), _ptr(input_ids), int(input_ids.dtype == torch.int64), _ptr(input_quals), n, row_stride,
            first.ctypes.data_as(C.POINTER(C.c_int32)), n_tokens.ctypes.data_as(C.POINTER(C.c_int32)), _ptr(out)))
        return out

    def forward_shared_prefix(self, input_ids, input_quals, first: np.ndarray, n_tokens: np.ndarray, n_pad: np.ndarray,
                              pad_token_id: int = 4, out=None):
        """forward_ragged(first, n_tokens) for rows that begin with n_pad[r] [PAD] tokens (quality 0), as the reference's
        collator pads a batch (tokenizer.py:71-87): the pad runs of all rows go through the model once per launch
        (`dc_forward_shared_prefix`).  Same logits, pad columns included."""
        n, row_stride = input_ids.shape
        first = np.ascontiguousarray(first, dtype=np.int32)
        n_tokens = np.ascontiguousarray(n_tokens, dtype=np.int32)
        n_pad = np.ascontiguousarray(n_pad, dtype=np.int32)
        assert first.shape == n_tokens.shape == n_pad.shape == (n,)
        if out is None:
            out = torch.zeros((n, row_stride, self.cfg.num_class), dtype=torch.float32, device=input_ids.device)
        i32p = C.POINTER(C.c_int32)
        _lib.check(_lib.lib().dc_forward_shared_prefix(
            self._h, _stream(), _ptr(input_ids), int(input_ids.dtype == torch.int64), _ptr(input_quals), n, row_stride,
            first.ctypes.data_as(i32p), n_tokens.ctypes.data_as(i32p), n_pad.ctypes.data_as(i32p), int(pad_token_id), _ptr(out)))
        return out

    def set_prefix_mode(self, mode: str) -> None:
        """How `forward_shared_prefix` shares the pad runs: "exact" (the long convolution still walks every row's padded
        sequence; bit-identical to the padded launch on the block-Toeplitz forms) or "linear" (y = (k * (z - z_pad) + F) * gate:
        the long convolution covers a row's own tokens only; equal to fp32 rounding)."""
        _lib.check(_lib.lib().dc_model_set_prefix_mode(self._h, {"exact": 1, "linear": 2}[mode]))
        self.prefix_mode = mode

    def prefix_violations(self) -> int:
        """Declared pad positions of `forward_shared_prefix` launches that did not hold ([PAD], 0.0) (synchronises)."""
        v = C.c_int32()
        _lib.check(_lib.lib().dc_model_prefix_violations(self._h, _stream(), C.byref(v)))
        return int(v.value)

    def head_forward(self, hidden: torch.Tensor, input_quals: torch.Tensor) -> torch.Tensor:
        """Diagnostic: final LayerNorm + head on a residual stream f32[B, L, d_model] -> logits f32[B, L, 2]."""
        assert hidden.dim() == 3 and hidden.shape[:2] == input_quals.shape and hidden.shape[2] == self.cfg.d_model
        assert hidden.dtype == torch.float32 and input_quals.dtype == torch.float32
        B, L, _ = hidden.shape
        out = torch.empty((B, L, self.cfg.num_class), dtype=torch.float32, device=hidden.device)
        _lib.check(_lib.lib().dc_head_forward(self._h, _stream(), _ptr(hidden), _ptr(input_quals), B, L, _ptr(out)))
        return out

    def forward_checked(self, input_ids, input_quals, first: np.ndarray | None = None, n_tokens: np.ndarray | None = None):
        """forward / forward_ragged with the fp16x3 range guard consulted: if an activation left the fp16 range
        the batch is re-run with the bf16 split (fp32 exponent range).  Synchronises the stream in fp16x3 mode;
        pipelined callers attribute the guard per batch themselves (`set_overflow_target`)."""
        run = (lambda: self.forward(input_ids, input_quals)) if first is None else (
            lambda: self.forward_ragged(input_ids, input_quals, first, n_tokens))
        if self.gemm_mode != "fp16x3":
            return run()
        counter = torch.zeros(1, dtype=torch.int32, device=input_ids.device)
        self.set_overflow_target(counter)
        try:
            out = run()
        finally:
            self.set_overflow_target(None)
        if int(counter.item()) > 0:
            self.set_gemm_mode("bf16x6")
            try:
                out = run()
            finally:
                self.set_gemm_mode("fp16x3")
        return out

    def set_overflow_target(self, counter: torch.Tensor | None):
        """Route the fp16x3 range guard of the forwards launched from now on into `counter` (int32[1] on the
        device, zeroed by the caller); None restores the handle's own counter."""
        if counter is not None:
            assert counter.is_cuda and counter.dtype == torch.int32 and counter.numel() >= 1
        _lib.check(_lib.lib().dc_model_set_overflow_target(self._h, _ptr(counter)))

    def filter(self, layer: int, seq_len: int) -> torch.Tensor:
        out = torch.empty((self.cfg.d_model, seq_len), dtype=torch.float32, device=_dev())
        _lib.check(_lib.lib().dc_model_filter(self._h, _stream(), layer, seq_len, _ptr(out)))
        return out

    def device_bytes(self) -> int:
        return int(_lib.lib().dc_model_device_bytes(self._h))

    def set_gemm_mode(self, mode: str):
        """"f32": fp32-input MFMA; "bf16x6": error-free 3-way bf16 split on bf16 MFMA (fp32-equivalent)."""
        _lib.check(_lib.lib().dc_model_set_gemm_mode(self._h, {"f32": 0, "bf16x6": 1, "fp16x3": 2}[mode]))
        self.gemm_mode = mode

    def set_fft_threshold(self, min_tokens: int):
        """Reads with more than `min_tokens` tokens take the O(L log L) FFT long convolution (default 2560)."""
        _lib.check(_lib.lib().dc_model_set_fft_threshold(self._h, int(min_tokens)))

    def set_fft_split(self, on: bool):
        """True (default): split / mixed-radix FFT size classes (3 passes, 3 x and 5 x 2^k points); False: the power-of-two
        transforms of rounds 2-4 (the A/B reference)."""
        _lib.check(_lib.lib().dc_model_set_fft_split(self._h, 1 if on else 0))

    def set_mlp_fusion(self, level):
        """fp16x3.  0 / False: fc1 and fc2 as two GEMM launches; 1: fc1 -> GELU -> fc2 as one kernel;
        2 / True (default): that kernel also runs the GEMM that consumes LayerNorm(its output) -- the next
        block's in_proj or the head's linear1."""
        lvl = 2 if level is True else int(level)
        _lib.check(_lib.lib().dc_model_set_mlp_fusion(self._h, lvl))

    def overflow(self) -> int:
        """fp16x3 range guard: workgroups that met an activation outside the fp16 range since the last call
        (synchronises the stream, clears the counter)."""
        n = C.c_int32()
        _lib.check(_lib.lib().dc_model_overflow(self._h, _stream(), C.byref(n)))
        return int(n.value)

    def set_profiling(self, on: bool):
        _lib.check(_lib.lib().dc_model_set_profiling(self._h, int(on)))

    def profile_reset(self):
        _lib.check(_lib.lib().dc_model_profile_reset(self._h))

    def profile(self) -> dict[str, tuple[float, int]]:
        """{stage: (total_ms, launches)} -- call after synchronising the stream."""
        buf = C.create_string_buffer(4096)
        _lib.check(_lib.lib().dc_model_profile_stages(self._h, buf, 4096))
        out = {}
        for name in filter(None, buf.value.decode().split(",")):
            ms, cnt = C.c_double(), C.c_int64()
            _lib.check(_lib.lib().dc_model_profile_get(self._h, name.encode(), C.byref(ms), C.byref(cnt)))
            out[name] = (ms.value, cnt.value)
        return out
