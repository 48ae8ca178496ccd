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
import struct

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


# The same layouts for struct.pack, which fills them several times as fast as ctypes does.
_ROPE = struct.Struct("8if4x6Q8q")
_ATTEND = struct.Struct("5Q4q4if4x3QqQq")
assert _ROPE.size == C.sizeof(RopeArgs) and _ATTEND.size == C.sizeof(Kv8Attend)



def _pack(fmt, *args):
    try:
        return fmt.pack(*args)
    except struct.error as e:
        raise ValueError(f"an argument is out of range: {e}") from None


_torch = _L = None
_types: dict = {}


def _lib():
    global _torch, _L, _stream
    if _L is None:
        import torch
        L = lib()
        P, I, L64 = C.c_void_p, C.c_int32, C.c_int64
        for name, res, args in [
            ("qtts_op_rope", I, [P, P]),
            ("qtts_rope_freqs", I, [I, I, C.c_double, C.c_double, C.c_double, C.c_double, C.c_double, C.POINTER(C.c_double),
                                    C.POINTER(C.c_float)]),
            ("qtts_kv8_check", I, [P, P, P, P, I, I]),
            ("qtts_op_kv8_append", I, [P, P, P, P, P, P, L64, L64, L64, L64, I, I, P]),
            ("qtts_op_kv8_read", I, [P, P, P, P, I, P, P, I, I, P]),
            ("qtts_kv8_attend_ws", L64, [P, P]),
            ("qtts_op_kv8_attend", I, [P, P, P]),
            ("qtts_op_kv8_evict", I, [P, P, P, P, I, P, L64, I, I, I, P, P, P, P]),
        ]:
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _types.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 30})
        _stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
        _torch, _L = torch, L
    return _L


def _refuse(what):
    raise ValueError(what)


def _check(ok):
    if not ok:
        raise ValueError(_L.qtts_create_error().decode())


def _int32(t, n, device, name):
    """The address of a contiguous int32 tensor [n] on GPU number `device`."""
    if t.dtype is not _torch.int32 or t.dim() != 1 or t.shape[0] != n or not t.is_cuda or t.get_device() != device or not t.is_contiguous():
        _refuse(f"{name}: a contiguous int32 tensor [{n}] on cuda:{device}")
    return t.data_ptr()


def _table(t, n, device, name):
    if (t.dtype is not _torch.int32 or t.dim() != 2 or t.shape[0] != n or t.shape[1] < 1 or not t.is_cuda or t.get_device() != device or
            not t.is_contiguous()):
        _refuse(f"{name}: a contiguous int32 tensor [{n}, columns] on cuda:{device}")
    return t.data_ptr()


def rope_freqs(rot: int, theta: float, scaling: str = "none", factor: float = 1.0, original_len: float = 4096.0, beta_fast: float = 32.0,
               beta_slow: float = 1.0, device=None):
    """(angles per position [rot/2] float64, factor on the rotated values) for `rope`.

    scaling: "none", "linear" (positions divided by factor), "ntk" (a larger base)
    or "yarn" (high-frequency dims kept, low ones divided, a ramp between, over a
    model trained on original_len positions).
    """
    L = _lib()
    if scaling not in SCALINGS:
        _refuse(f"scaling is one of {', '.join(SCALINGS)}")
    if not isinstance(rot, int) or not 2 <= rot <= 4096:
        _refuse("rot is even, 2 to 4096")
    f = (C.c_double * (rot // 2))()
    m = C.c_float(1.0)
    _check(L.qtts_rope_freqs(SCALINGS[scaling], rot, theta, factor, original_len, beta_fast, beta_slow, f, C.byref(m)))
    return _torch.tensor(list(f), dtype=_torch.float64, device=device), m.value


def rope(q, k, positions, freq, *, layout: str = "half", factor: float = 1.0, q_out=None, k_out=None):
    """Turns the first 2 * len(freq) dims of every head of q [T, heads, dim] and
    k [T, kv_heads, dim] (k None: q alone) by positions [T] (int32) times freq
    (float64, radians); layout "half" pairs dims (i, i + rot/2), "interleaved" (2i,
    2i + 1).  float16, bfloat16 or float32; heads may be strided, dims contiguous.
    Returns (q, k) rotated: new tensors, or q_out / k_out, which may be q and k.
    """
    L = _L or _lib()
    if not q.is_cuda or q.dim() != 3 or q.dtype not in _types:
        _refuse("q: a CUDA tensor [T, heads, dim] of float16, bfloat16 or float32")
    T, heads, dim = q.shape
    dev, ty = q.get_device(), q.dtype
    qr, qh, qd = q.stride()
    if qd != 1:
        _refuse("q: the dims of a head are contiguous")
    if layout != "half" and layout != "interleaved":
        _refuse("layout is 'half' or 'interleaved'")
    if freq.dtype is not _torch.float64 or freq.dim() != 1 or not freq.is_cuda or freq.get_device() != dev or not freq.is_contiguous():
        _refuse("freq: a contiguous float64 tensor on q's device")
    pos = _int32(positions, T, dev, "positions")
    if q_out is None:
        q_out = _torch.empty((T, heads, dim), dtype=ty, device=q.device)
        qor, qoh = heads * dim, dim
    else:
        if q_out.shape != q.shape or q_out.dtype is not ty or q_out.device != q.device or q_out.stride(2) != 1:
            _refuse("q_out is like q")
        qor, qoh = q_out.stride(0), q_out.stride(1)
    kh = kp = kop = kr = kd = kor = kod = 0
    if k is not None:
        if k.dim() != 3 or k.shape[0] != T or k.shape[2] != dim or k.dtype is not ty or not k.is_cuda or k.get_device() != dev or k.stride(2) != 1:
            _refuse("k: [T, kv_heads, dim] like q")
        kh = k.shape[1]
        if k_out is None:
            k_out = _torch.empty((T, kh, dim), dtype=ty, device=k.device)
        elif k_out.shape != k.shape or k_out.dtype is not ty or k_out.device != k.device or k_out.stride(2) != 1:
            _refuse("k_out is like k")
        if kh:
            kp, kop = k.data_ptr(), k_out.data_ptr()
            kr, kd, _ = k.stride()
            kor, kod, _ = k_out.stride()
    if T:
        _check(L.qtts_op_rope(_pack(_ROPE, dev, _types[ty], T, heads, kh, dim, 2 * freq.shape[0], layout == "interleaved", factor, pos, freq.data_ptr(),
                                         q.data_ptr(), kp, q_out.data_ptr(), kop, qr, qh, kr, kd, qor, qoh, kor, kod), _stream(dev)))
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
        if not k.is_cuda or k.dim() != 4 or k.shape[2] != PAGE or k.shape[3] not in (64, 128, 256) or k.dtype not in (t.int8, t.float8_e4m3fn):
            _refuse("k: a CUDA tensor [pages, kv_heads, 64, dim] of int8 or float8_e4m3fn codes, dim 64, 128 or 256")
        P, H, _, D = k.shape
        if v.shape != k.shape or v.dtype is not k.dtype:
            _refuse("v is like k")
        for n, x in (("k_scale", k_scale), ("v_scale", v_scale)):
            if x.dtype is not t.float32 or x.shape != (P, H, PAGE // BLOCK):
                _refuse(f"{n}: float32 [pages, kv_heads, 4]")
        if k_open.dtype not in (t.float16, t.bfloat16) or k_open.dim() != 4 or k_open.shape[1:] != (H, RING, D):
            _refuse("k_open: float16 or bfloat16 [seqs, kv_heads, 32, dim]")
        if v_open.shape != k_open.shape or v_open.dtype is not k_open.dtype:
            _refuse("v_open is like k_open")
        if status is None:
            status = t.zeros(1, dtype=t.int32, device=k.device)
        if status.dtype is not t.int32 or status.numel() != 1:
            _refuse("status: one int32")
        for x in (v, k_scale, v_scale, k_open, v_open, status):
            if x.device != k.device:
                _refuse("the cache's tensors are on one device")
        for x in (k, v, k_scale, v_scale, k_open, v_open):
            if not x.is_contiguous():
                _refuse("the cache's tensors are contiguous")
        self.k, self.v, self.k_scale, self.v_scale, self.k_open, self.v_open, self.status = k, v, k_scale, v_scale, k_open, v_open, status
        self.device, self.row_type, self.seqs, self.kv_heads, self.dim, self.pages = k.device, k_open.dtype, k_open.shape[0], H, D, P
        self._dev = k.get_device()
        self._head = (self._dev, int(k.dtype is t.float8_e4m3fn), _types[k_open.dtype], H, D, P, k_open.shape[0])
        self._ptrs = tuple(x.data_ptr() for x in (k, v, k_scale, v_scale, k_open, v_open, status))
        self._c = {}                       # the C descriptor for each number of columns that page tables have had

    @classmethod
    def empty(cls, pages: int, seqs: int, kv_heads: int, dim: int, *, code: str = "int8", dtype=None, device="cuda"):
        """A cache with memory of its own: code "int8" or "e4m3", dtype torch.float16 (default) or torch.bfloat16."""
        import torch
        if code not in ("int8", "e4m3"):
            _refuse("code is 'int8' or 'e4m3'")
        d = torch.device(device)
        if d.type == "cuda" and d.index is None:
            d = torch.device("cuda", torch.cuda.current_device())
        c = torch.int8 if code == "int8" else torch.float8_e4m3fn
        codes = [torch.zeros(pages, kv_heads, PAGE, dim, dtype=torch.uint8, device=d).view(c) for _ in range(2)]
        scales = [torch.zeros(pages, kv_heads, PAGE // BLOCK, dtype=torch.float32, device=d) for _ in range(2)]
        rings = [torch.zeros(seqs, kv_heads, RING, dim, dtype=dtype or torch.float16, device=d) for _ in range(2)]
        return cls(*codes, *scales, *rings)

    def _desc(self, columns):
        c = self._c.get(columns)
        if c is None:
            d = Kv8(*self._head, columns, *self._ptrs)
            c = self._c[columns] = (C.addressof(d), d)
        return c[0]

    def _packed(self, x, heads, name):
        if x.dim() != 3 or x.shape[2] != self.dim or x.shape[1] != heads or x.dtype is not self.row_type or not x.is_cuda or \
                x.get_device() != self._dev or x.stride(2) != 1:
            _refuse(f"{name}: [rows, {heads}, {self.dim}] {self.row_type} on {self.device}, dims contiguous")

    def _cu(self, cu, rows, most, what):
        if cu is None:
            if rows != self.seqs:
                _refuse("without cu there is one row for each sequence")
            return None, 1
        if most is None or most < 0:
            _refuse(f"{what}: the most rows of one sequence")
        return _int32(cu, self.seqs + 1, self._dev, "cu"), most

    def _weight(self, w, table, name):
        if w.dtype is not _torch.float32 or w.dim() != 3 or w.shape[0] != self.seqs or w.shape[1] != self.kv_heads or \
                w.shape[2] < table.shape[1] * PAGE or not w.is_contiguous() or not w.is_cuda or w.get_device() != self._dev:
            _refuse(f"{name}: a contiguous float32 tensor [seqs, kv_heads, >= 64 columns of table]")
        return w.data_ptr()

    def append(self, k, v, table, lens, cu=None, max_new: int | None = None) -> None:
        """The packed rows k, v [T, kv_heads, dim] become the last ones of their
        sequences; lens are the lengths AFTER them.  max_new: the most rows that one
        sequence brings (needed with cu)."""
        tp = _table(table, self.seqs, self._dev, "table")
        self._packed(k, self.kv_heads, "k")
        self._packed(v, self.kv_heads, "v")
        T = k.shape[0]
        if v.shape[0] != T:
            _refuse("v is like k")
        cu_p, most = self._cu(cu, T, max_new, "max_new")
        kr, kh, _ = k.stride()
        vr, vh, _ = v.stride()
        _check(_L.qtts_op_kv8_append(self._desc(table.shape[1]), tp, _int32(lens, self.seqs, self._dev, "lens"), cu_p, k.data_ptr(), v.data_ptr(),
                                     kr, kh, vr, vh, T, most, _stream(self._dev)))

    def read(self, table, begin, cu, rows: int, max_rows: int, dtype=None):
        """(k, v) [rows, kv_heads, dim] of dtype (default the rows' type): cu[b+1] - cu[b]
        rows of sequence b from position begin[b] (None: 0) on, packed; max_rows: the
        most of one sequence.  Rows that belong to no sequence are not written."""
        tp = _table(table, self.seqs, self._dev, "table")
        dtype = dtype or self.row_type
        if dtype not in _types:
            _refuse("dtype is float32, float16 or bfloat16")
        if rows < 0:
            _refuse("rows")
        cu_p, most = self._cu(cu, rows, max_rows, "max_rows")
        bp = None if begin is None else _int32(begin, self.seqs, self._dev, "begin")
        shape = (rows, self.kv_heads, self.dim)
        k, v = _torch.empty(shape, dtype=dtype, device=self.device), _torch.empty(shape, dtype=dtype, device=self.device)
        _check(_L.qtts_op_kv8_read(self._desc(table.shape[1]), tp, bp, cu_p, _types[dtype], k.data_ptr(), v.data_ptr(), rows, most,
                                   _stream(self._dev)))
        return k, v

    def attend(self, q, table, lens, cu=None, max_q: int | None = None, *, scale: float, window: int = 0, weight=None, weight_out=None,
               want_lse: bool = False, out=None):
        """Causal attention of q [T, heads, dim] over the cache: (out like q, lse [T, heads]
        float32 or None).  The rows of a sequence are its last positions (append them
        first); with window > 0 a row sees that many keys, itself included.  weight,
        weight_out [seqs, kv_heads, >= 64 columns] float32, contiguous:
        weight_out = weight + each key's softmax weights over the head group and the
        rows (weight_out None: in place)."""
        tp = _table(table, self.seqs, self._dev, "table")
        if q.dim() != 3:
            _refuse("q: [rows, heads, dim]")
        T, heads, _ = q.shape
        self._packed(q, heads, "q")
        if heads < 1 or heads % self.kv_heads:
            _refuse("heads is a multiple of kv_heads")
        cu_p, most = self._cu(cu, T, max_q, "max_q")
        if out is None:
            out = _torch.empty((T, heads, self.dim), dtype=self.row_type, device=self.device)
        else:
            self._packed(out, heads, "out")
            if out.shape[0] != T:
                _refuse("out is like q")
        lse = _torch.empty((T, heads), dtype=_torch.float32, device=self.device) if want_lse else None
        wi = wo = ws = 0
        if weight is not None:
            weight_out = weight if weight_out is None else weight_out
            wi, wo, ws = self._weight(weight, table, "weight"), self._weight(weight_out, table, "weight_out"), weight.shape[2]
            if weight_out.shape != weight.shape:
                _refuse("weight_out is like weight")
        elif weight_out is not None:
            _refuse("weight_out goes with weight")
        c = self._desc(table.shape[1])
        qr, qh, _ = q.stride()
        orow, oh, _ = out.stride()
        args = (tp, _int32(lens, self.seqs, self._dev, "lens"), cu_p or 0, q.data_ptr(), out.data_ptr(), qr, qh, orow, oh, T, most, heads, window, scale,
                0 if lse is None else lse.data_ptr(), wi, wo, ws)
        a = _pack(_ATTEND, *args, 0, 0)
        n = _L.qtts_kv8_attend_ws(c, a)
        if n > 0:
            space = _torch.empty(n, dtype=_torch.uint8, device=self.device)   # the stream's (or the graph's) own
            a = _pack(_ATTEND, *args, space.data_ptr(), n)
        _check(_L.qtts_op_kv8_attend(c, a, _stream(self._dev)))
        return out, lse

    def evict(self, table, lens, dst_table, weight, budget: int, *, sinks: int = 0, recent: int = 0):
        """Sequences longer than budget (a multiple of 16) keep, per kv head, their first
        `sinks` and last `recent` rows and the heaviest others by weight [seqs, kv_heads,
        >= 64 columns]; the rest keep all.  The kept rows move to the pages of dst_table
        [seqs, columns], which nothing else may use; the old pages are free afterwards.
        Returns (lens, keep [seqs, kv_heads, budget] positions, -1 past the end, weight
        of the kept)."""
        tp = _table(table, self.seqs, self._dev, "table")
        dp = _table(dst_table, self.seqs, self._dev, "dst_table")
        wp = self._weight(weight, table, "weight")
        if budget < 1:
            _refuse("budget is a multiple of 16")
        lens_out = _torch.empty(self.seqs, dtype=_torch.int32, device=self.device)
        keep = _torch.empty((self.seqs, self.kv_heads, budget), dtype=_torch.int32, device=self.device)
        weight_out = _torch.empty((self.seqs, self.kv_heads, budget), dtype=_torch.float32, device=self.device)
        _check(_L.qtts_op_kv8_evict(self._desc(table.shape[1]), tp, _int32(lens, self.seqs, self._dev, "lens"), dp, dst_table.shape[1], wp,
                                    weight.shape[2], budget, sinks, recent, lens_out.data_ptr(), keep.data_ptr(), weight_out.data_ptr(),
                                    _stream(self._dev)))
        return lens_out, keep, weight_out

    def check(self) -> None:
        """Waits for the device and raises if a kernel found a page, length or row that
        did not fit since the last check (it left that part out)."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise RuntimeError("kv cache: " + ", ".join(t for b, t in STATUS.items() if bits & b))
