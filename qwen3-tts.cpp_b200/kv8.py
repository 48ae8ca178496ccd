"""Rotary positions and the 8-bit paged key/value cache on torch CUDA tensors
(qtts_op_rope, qtts_op_kv8_* of include/qwen3tts_b200.h).

A decode step of a serving loop is `rope` on the projected heads,
`KvCache8.append` of the new rows, `KvCache8.attend` of the queries, and now and
then `KvCache8.evict` when the sequences have outgrown their budget.  Page tables
and lengths are the caller's int32 tensors, so the calls never synchronise, can
be captured into CUDA graphs, and run on the current stream of the tensors'
device.  Arguments that do not fit raise ValueError before anything is launched;
page numbers and lengths live on the device and are checked there
(`KvCache8.check`).
"""
from __future__ import annotations

import ctypes as C

from .engine import lib

PAGE, BLOCK, RING = 64, 16, 32
SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}
STATUS = {1: "a page number outside the pool", 2: "a length outside the page table", 4: "rows outside the call's tensors",
          8: "a destination page that is in use", 16: "a copy that did not arrive in time"}


class RopeArgs(C.Structure):
    _fields_ = [("device", C.c_int32), ("type", C.c_int32), ("rows", C.c_int32), ("q_heads", C.c_int32), ("k_heads", C.c_int32),
                ("dim", C.c_int32), ("rot", C.c_int32), ("interleaved", C.c_int32), ("factor", C.c_float),
                ("pos", C.c_void_p), ("freq", C.c_void_p), ("q", C.c_void_p), ("k", C.c_void_p), ("q_out", C.c_void_p),
                ("k_out", C.c_void_p)] + [(n, C.c_int64) for n in ("q_row", "q_head", "k_row", "k_head", "qo_row", "qo_head",
                                                                   "ko_row", "ko_head")]


class Kv8(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("device", "code", "row_type", "n_kv_heads", "head_dim", "n_pages", "n_seqs", "max_pages")] + [
        (n, C.c_void_p) for n in ("k", "v", "k_scale", "v_scale", "k_open", "v_open", "status")]


class Kv8Attend(C.Structure):
    _fields_ = [("table", C.c_void_p), ("lens", C.c_void_p), ("cu", C.c_void_p), ("q", C.c_void_p), ("out", C.c_void_p)] + [
        (n, C.c_int64) for n in ("q_row", "q_head", "o_row", "o_head")] + [
        (n, C.c_int32) for n in ("n_rows", "max_q", "n_heads", "window")] + [
        ("scale", C.c_float), ("lse", C.c_void_p), ("weight_in", C.c_void_p), ("weight_out", C.c_void_p), ("weight_stride", C.c_int64),
        ("ws", C.c_void_p), ("ws_bytes", C.c_int64)]


_sig_done = False
_torch = None
_types: dict = {}


def _lib():
    global _sig_done, _torch
    L = lib()
    if not _sig_done:
        import torch
        P, I, L64 = C.c_void_p, C.c_int32, C.c_int64
        for name, res, args in [
            ("qtts_op_rope", I, [C.POINTER(RopeArgs), P]),
            ("qtts_rope_freqs", I, [I, I, C.c_double, C.c_double, C.c_double, C.c_double, C.c_double, C.POINTER(C.c_double),
                                    C.POINTER(C.c_float)]),
            ("qtts_kv8_check", I, [C.POINTER(Kv8), P, P, P, I, I]),
            ("qtts_op_kv8_append", I, [C.POINTER(Kv8), P, P, P, P, P, L64, L64, L64, L64, I, I, P]),
            ("qtts_op_kv8_read", I, [C.POINTER(Kv8), P, P, P, I, P, P, I, I, P]),
            ("qtts_kv8_attend_ws", L64, [C.POINTER(Kv8), C.POINTER(Kv8Attend)]),
            ("qtts_op_kv8_attend", I, [C.POINTER(Kv8), C.POINTER(Kv8Attend), P]),
            ("qtts_op_kv8_evict", I, [C.POINTER(Kv8), P, P, P, I, P, L64, I, I, I, P, P, P, P]),
        ]:
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _torch = torch
        _types.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 30})
        _sig_done = True
    return L


def _refused(ok):
    if not ok:
        raise ValueError(lib().qtts_create_error().decode())


def _need(cond, what):
    if not cond:
        raise ValueError(what)


def _int32(t, shape, device, name):
    _need(t.dtype is _torch.int32 and t.shape == shape and t.device == device and t.is_contiguous(),
          f"{name}: a contiguous int32 tensor of shape {tuple(shape)} on {device}")
    return t.data_ptr()


def _stream(device):
    return _torch.cuda.current_stream(device).cuda_stream


def _is_cuda(t, name):
    _need(t.is_cuda, f"{name}: a CUDA tensor")


def rope_freqs(rot: int, theta: float, scaling: str = "none", factor: float = 1.0, original_len: float = 4096.0, beta_fast: float = 32.0,
               beta_slow: float = 1.0, device=None):
    """(angles per position [rot/2] float64, factor on the rotated values) for `rope`.

    scaling: "none", "linear" (positions divided by factor), "ntk" (a larger base)
    or "yarn" (high-frequency dims kept, low ones divided, a ramp between, over a
    model trained on original_len positions).
    """
    L = _lib()
    _need(scaling in SCALINGS, f"scaling is one of {', '.join(SCALINGS)}")
    _need(isinstance(rot, int) and 2 <= rot <= 4096, "rot is even, 2 to 4096")
    f = (C.c_double * (rot // 2))()
    m = C.c_float(1.0)
    _refused(L.qtts_rope_freqs(SCALINGS[scaling], rot, theta, factor, original_len, beta_fast, beta_slow, f, C.byref(m)))
    return _torch.tensor(list(f), dtype=_torch.float64, device=device), m.value


def rope(q, k, positions, freq, *, layout: str = "half", factor: float = 1.0, q_out=None, k_out=None):
    """Turns the first 2 * len(freq) dims of every head of q [T, heads, dim] and
    k [T, kv_heads, dim] (k None: q alone) by positions [T] (int32) times freq
    (float64, radians); layout "half" pairs dims (i, i + rot/2), "interleaved" (2i,
    2i + 1).  float16, bfloat16 or float32; heads may be strided, dims contiguous.
    Returns (q, k) rotated: new tensors, or q_out / k_out, which may be q and k.
    """
    L = _lib()
    _is_cuda(q, "q")
    _need(layout in ("half", "interleaved"), "layout is 'half' or 'interleaved'")
    _need(q.dtype in _types and q.dim() == 3 and (q.shape[2] == 0 or q.stride(2) == 1), "q: [T, heads, dim] of float16, bfloat16 or float32, dims contiguous")
    T, heads, dim = q.shape
    _int32(positions, (T,), q.device, "positions")
    _need(freq.dtype is _torch.float64 and freq.dim() == 1 and freq.is_contiguous() and freq.device == q.device,
          "freq: a contiguous float64 tensor on q's device")
    if q_out is None:
        q_out = _torch.empty((T, heads, dim), dtype=q.dtype, device=q.device)
    else:
        _need(q_out.shape == q.shape and q_out.dtype is q.dtype and q_out.device == q.device and q_out.stride(2) == 1, "q_out is like q")
    a = RopeArgs(q.device.index, _types[q.dtype], T, heads, 0, dim, 2 * freq.shape[0], layout == "interleaved", factor,
                 positions.data_ptr(), freq.data_ptr(), q.data_ptr(), None, q_out.data_ptr(), None,
                 q.stride(0), q.stride(1), 0, 0, q_out.stride(0), q_out.stride(1), 0, 0)
    if k is not None:
        _need(k.dim() == 3 and k.shape[0] == T and k.shape[2] == dim and k.dtype is q.dtype and k.device == q.device and k.stride(2) == 1,
              "k: [T, kv_heads, dim] like q")
        if k_out is None:
            k_out = _torch.empty((T, k.shape[1], dim), dtype=q.dtype, device=q.device)
        else:
            _need(k_out.shape == k.shape and k_out.dtype is k.dtype and k_out.device == k.device and k_out.stride(2) == 1, "k_out is like k")
        if k.shape[1]:
            a.k_heads, a.k, a.k_out = k.shape[1], k.data_ptr(), k_out.data_ptr()
            a.k_row, a.k_head, a.ko_row, a.ko_head = k.stride(0), k.stride(1), k_out.stride(0), k_out.stride(1)
    if T:
        _refused(L.qtts_op_rope(C.byref(a), _stream(q.device)))
    return q_out, k_out


class KvCache8:
    """A handle on the caller's 8-bit cache pool.

    k, v [pages, kv_heads, 64, dim]: codes, torch.int8 or torch.float8_e4m3fn;
    k_scale, v_scale [pages, kv_heads, 4] float32: one scale per 16 tokens;
    k_open, v_open [seqs, kv_heads, 32, dim] float16 or bfloat16: the rows of each
    sequence's last two blocks.  All contiguous, on one device; dim 64, 128 or 256.
    `KvCache8.empty` allocates them.

    Calls take `table` [seqs, columns] (pages of each sequence in order) and `lens`
    [seqs], int32.  `cu` [seqs + 1] int32 gives each sequence's rows of the packed
    tensors (None: one row each).  Two calls in flight at once on different streams
    must not write the same pages, rings or outputs.
    """

    def __init__(self, k, v, k_scale, v_scale, k_open, v_open, status=None):
        _lib()
        t = _torch
        _is_cuda(k, "k")
        _need(k.dim() == 4 and k.shape[2] == PAGE and k.shape[3] in (64, 128, 256), "k: [pages, kv_heads, 64, dim], dim 64, 128 or 256")
        _need(k.dtype in (t.int8, t.float8_e4m3fn), "k: torch.int8 or torch.float8_e4m3fn codes")
        P, H, _, D = k.shape
        _need(v.shape == k.shape and v.dtype is k.dtype, "v is like k")
        for n, s in (("k_scale", k_scale), ("v_scale", v_scale)):
            _need(s.dtype is t.float32 and s.shape == (P, H, PAGE // BLOCK), f"{n}: float32 [pages, kv_heads, 4]")
        _need(k_open.dtype in (t.float16, t.bfloat16) and k_open.dim() == 4 and k_open.shape[1:] == (H, RING, D),
              "k_open: float16 or bfloat16 [seqs, kv_heads, 32, dim]")
        _need(v_open.shape == k_open.shape and v_open.dtype is k_open.dtype, "v_open is like k_open")
        if status is None:
            status = t.zeros(1, dtype=t.int32, device=k.device)
        _need(status.dtype is t.int32 and status.numel() == 1, "status: one int32")
        for x in (v, k_scale, v_scale, k_open, v_open, status):
            _need(x.device == k.device, "the cache's tensors are on one device")
        for x in (k, v, k_scale, v_scale, k_open, v_open):
            _need(x.is_contiguous(), "the cache's tensors are contiguous")
        self.k, self.v, self.k_scale, self.v_scale, self.k_open, self.v_open, self.status = k, v, k_scale, v_scale, k_open, v_open, status
        self.device, self.row_type, self.seqs, self.kv_heads, self.dim, self.pages = k.device, k_open.dtype, k_open.shape[0], H, D, P
        self._dims = (k.device.index, int(k.dtype is t.float8_e4m3fn), _types[k_open.dtype], H, D, P, k_open.shape[0])
        self._ptrs = tuple(x.data_ptr() for x in (k, v, k_scale, v_scale, k_open, v_open, status))

    @classmethod
    def empty(cls, pages: int, seqs: int, kv_heads: int, dim: int, *, code: str = "int8", dtype=None, device="cuda"):
        """A cache with memory of its own: code "int8" or "e4m3", dtype torch.float16 (default) or torch.bfloat16."""
        import torch
        _need(code in ("int8", "e4m3"), "code is 'int8' or 'e4m3'")
        d = torch.device(device)
        if d.type == "cuda" and d.index is None:
            d = torch.device("cuda", torch.cuda.current_device())
        c = torch.int8 if code == "int8" else torch.float8_e4m3fn
        codes = [torch.zeros(pages, kv_heads, PAGE, dim, dtype=torch.uint8, device=d).view(c) for _ in range(2)]
        scales = [torch.zeros(pages, kv_heads, PAGE // BLOCK, dtype=torch.float32, device=d) for _ in range(2)]
        rings = [torch.zeros(seqs, kv_heads, RING, dim, dtype=dtype or torch.float16, device=d) for _ in range(2)]
        return cls(*codes, *scales, *rings)

    def _desc(self, table):
        _need(table.dtype is _torch.int32 and table.dim() == 2 and table.shape[0] == self.seqs and table.shape[1] > 0 and
              table.is_contiguous() and table.device == self.device,
              f"table: a contiguous int32 tensor [{self.seqs}, columns] on {self.device}")
        return Kv8(*self._dims, table.shape[1], *self._ptrs)

    def _packed(self, x, heads, name):
        _need(x.dim() == 3 and x.shape[2] == self.dim and (heads is None or x.shape[1] == heads) and x.dtype is self.row_type and
              x.device == self.device and x.stride(2) == 1,
              f"{name}: [rows, {heads or 'heads'}, {self.dim}] {self.row_type} on {self.device}, dims contiguous")

    def _cu(self, cu, rows, most, what):
        if cu is None:
            _need(rows == self.seqs, "without cu there is one row for each sequence")
            return None, 1
        _need(most is not None and most >= 0, f"{what}: the most rows of one sequence")
        return _int32(cu, (self.seqs + 1,), self.device, "cu"), most

    def append(self, k, v, table, lens, cu=None, max_new: int | None = None) -> None:
        """The packed rows k, v [T, kv_heads, dim] become the last ones of their
        sequences; lens are the lengths AFTER them.  max_new: the most rows that one
        sequence brings (needed with cu)."""
        c = self._desc(table)
        self._packed(k, self.kv_heads, "k")
        self._packed(v, self.kv_heads, "v")
        _need(v.shape == k.shape, "v is like k")
        cu_p, most = self._cu(cu, k.shape[0], max_new, "max_new")
        _refused(lib().qtts_op_kv8_append(C.byref(c), table.data_ptr(), _int32(lens, (self.seqs,), self.device, "lens"), cu_p, k.data_ptr(),
                                          v.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1), k.shape[0], most,
                                          _stream(self.device)))

    def read(self, table, begin, cu, rows: int, max_rows: int, dtype=None):
        """(k, v) [rows, kv_heads, dim] of dtype (default the rows' type): cu[b+1] - cu[b]
        rows of sequence b from position begin[b] (None: 0) on, packed; max_rows: the
        most of one sequence.  Rows that belong to no sequence are not written."""
        c = self._desc(table)
        dtype = dtype or self.row_type
        _need(dtype in _types, "dtype is float32, float16 or bfloat16")
        _need(rows >= 0, "rows")
        cu_p, most = self._cu(cu, rows, max_rows, "max_rows")
        bp = None if begin is None else _int32(begin, (self.seqs,), self.device, "begin")
        k, v = (_torch.empty(rows, self.kv_heads, self.dim, dtype=dtype, device=self.device) for _ in range(2))
        _refused(lib().qtts_op_kv8_read(C.byref(c), table.data_ptr(), bp, cu_p, _types[dtype], k.data_ptr(), v.data_ptr(), rows, most,
                                        _stream(self.device)))
        return k, v

    def attend(self, q, table, lens, cu=None, max_q: int | None = None, *, scale: float, window: int = 0, weight=None, weight_out=None,
               want_lse: bool = False, out=None):
        """Causal attention of q [T, heads, dim] over the cache: (out like q, lse [T, heads]
        float32 or None).  The rows of a sequence are its last positions (append them
        first); with window > 0 a row sees that many keys, itself included.  weight,
        weight_out [seqs, kv_heads, >= 64 columns] float32, dims contiguous:
        weight_out = weight + each key's softmax weights over the head group and the
        rows (weight_out None: in place)."""
        c = self._desc(table)
        self._packed(q, None, "q")
        T, heads, _ = q.shape
        _need(heads > 0 and heads % self.kv_heads == 0, "heads is a multiple of kv_heads")
        cu_p, most = self._cu(cu, T, max_q, "max_q")
        if out is None:
            out = _torch.empty((T, heads, self.dim), dtype=q.dtype, device=self.device)
        else:
            self._packed(out, heads, "out")
            _need(out.shape == q.shape, "out is like q")
        lse = _torch.empty((T, heads), dtype=_torch.float32, device=self.device) if want_lse else None
        a = Kv8Attend(table.data_ptr(), _int32(lens, (self.seqs,), self.device, "lens"), cu_p, q.data_ptr(), out.data_ptr(),
                      q.stride(0), q.stride(1), out.stride(0), out.stride(1), T, most, heads, window, scale,
                      None if lse is None else lse.data_ptr())
        if weight is not None:
            weight_out = weight if weight_out is None else weight_out
            for n, w in (("weight", weight), ("weight_out", weight_out)):
                _need(w.dtype is _torch.float32 and w.dim() == 3 and w.shape[:2] == (self.seqs, self.kv_heads) and w.shape[2] >= table.shape[1] * PAGE and
                      w.is_contiguous() and w.device == self.device, f"{n}: a contiguous float32 tensor [seqs, kv_heads, >= 64 columns of table]")
            _need(weight_out.shape == weight.shape, "weight_out is like weight")
            a.weight_in, a.weight_out, a.weight_stride = weight.data_ptr(), weight_out.data_ptr(), weight.shape[2]
        else:
            _need(weight_out is None, "weight_out goes with weight")
        L = lib()
        n = L.qtts_kv8_attend_ws(C.byref(c), C.byref(a))
        if n > 0:
            ws = _torch.empty(n, dtype=_torch.uint8, device=self.device)   # the stream's (or the graph's) own
            a.ws, a.ws_bytes = ws.data_ptr(), n
        _refused(L.qtts_op_kv8_attend(C.byref(c), C.byref(a), _stream(self.device)))
        return out, lse

    def evict(self, table, lens, dst_table, weight, budget: int, *, sinks: int = 0, recent: int = 0):
        """Sequences longer than budget (a multiple of 16) keep, per kv head, their first
        `sinks` and last `recent` rows and the heaviest others by weight [seqs, kv_heads,
        >= 64 columns]; the rest keep all.  The kept rows move to the pages of dst_table
        [seqs, columns], which nothing else may use; the old pages are free afterwards.
        Returns (lens, keep [seqs, kv_heads, budget] positions, -1 past the end, weight
        of the kept)."""
        c = self._desc(table)
        _need(dst_table.dtype is _torch.int32 and dst_table.dim() == 2 and dst_table.shape[0] == self.seqs and dst_table.is_contiguous() and
              dst_table.device == self.device, f"dst_table: a contiguous int32 tensor [{self.seqs}, columns] on {self.device}")
        _need(weight.dtype is _torch.float32 and weight.dim() == 3 and weight.shape[:2] == (self.seqs, self.kv_heads) and
              weight.shape[2] >= table.shape[1] * PAGE and weight.is_contiguous() and weight.device == self.device,
              "weight: a contiguous float32 tensor [seqs, kv_heads, >= 64 columns of table]")
        _need(budget > 0, "budget is a multiple of 16")
        lens_out = _torch.empty(self.seqs, dtype=_torch.int32, device=self.device)
        keep = _torch.empty((self.seqs, self.kv_heads, budget), dtype=_torch.int32, device=self.device)
        weight_out = _torch.empty((self.seqs, self.kv_heads, budget), dtype=_torch.float32, device=self.device)
        _refused(lib().qtts_op_kv8_evict(C.byref(c), table.data_ptr(), _int32(lens, (self.seqs,), self.device, "lens"), dst_table.data_ptr(),
                                         dst_table.shape[1], weight.data_ptr(), weight.shape[2], budget, sinks, recent, lens_out.data_ptr(),
                                         keep.data_ptr(), weight_out.data_ptr(), _stream(self.device)))
        return lens_out, keep, weight_out

    def check(self) -> None:
        """Waits for the device and raises if a kernel found a page, length or row that
        did not fit since the last check (it left that part out)."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise RuntimeError("kv cache: " + ", ".join(t for b, t in STATUS.items() if bits & b))
