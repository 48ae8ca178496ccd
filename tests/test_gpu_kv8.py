"""The rotary and 8-bit-cache operators on a B200 against plain float64 statements
(tests/kv8_ref.py).  Quantised values are compared bit for bit: their definition
is a fixed sequence of IEEE float32 steps.  Tolerances of the others are derived
beside the plain statements."""
from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

import kv8_ref as ref

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def kv8(qtts):
    import qtts_b200.kv8 as m
    return m


def rows(g, n, H, D, dtype):
    """Rows with a few channels several times as large as the rest."""
    x = torch.randn(n, H, D, generator=g)
    x[..., ::17] *= 7
    return x.to(dtype)


class Both:
    """A cache on the GPU and what it should hold."""

    def __init__(self, kv8, seqs, H, D, code, dtype, cols, spare=0, seed=0, device="cuda"):
        self.g = torch.Generator().manual_seed(seed)
        self.H, self.D, self.dtype, self.code, self.seqs, self.cols = H, D, dtype, code, seqs, cols
        self.cache = kv8.KvCache8.empty(seqs * cols + spare, seqs, H, D, code=code, dtype=dtype, device=device)
        # pages start with every bit set: NaN for e4m3 codes and for scales
        for t in (self.cache.k, self.cache.v):
            t.view(torch.uint8).fill_(255)
        self.cache.k_scale.fill_(math.nan)
        self.cache.v_scale.fill_(math.nan)
        self.cache.k_open.fill_(math.nan)
        self.cache.v_open.fill_(math.nan)
        order = torch.randperm(seqs * cols + spare, generator=self.g).to(torch.int32)
        self.table = order[: seqs * cols].reshape(seqs, cols).contiguous().to(device)
        self.spare = order[seqs * cols:].to(device)
        self.model = ref.Model(seqs, H, D, code, dtype)
        self.device = device

    def lens(self):
        return torch.tensor([r.shape[0] for r in self.model.rows[0]], dtype=torch.int32, device=self.device)

    def cu(self, counts):
        return torch.tensor([0] + list(counts), dtype=torch.int64).cumsum(0).to(torch.int32).to(self.device)

    def append(self, counts, k=None, v=None):
        k = rows(self.g, sum(counts), self.H, self.D, self.dtype) if k is None else k
        v = rows(self.g, sum(counts), self.H, self.D, self.dtype) if v is None else v
        at = 0
        for b, n in enumerate(counts):
            self.model.append(b, k[at: at + n], v[at: at + n])
            at += n
        one = all(n == 1 for n in counts)
        self.cache.append(k.to(self.device), v.to(self.device), self.table, self.lens(), None if one else self.cu(counts), None if one else max(counts))

    def read(self, dtype=torch.float32, table=None):
        counts = [r.shape[0] for r in self.model.rows[0]]
        k, v = self.cache.read(self.table if table is None else table, None, self.cu(counts), sum(counts), max(counts), dtype)
        return [x.cpu().split(counts) for x in (k, v)]

    def same(self):
        got = self.read()
        for side in range(2):
            for b in range(self.seqs):
                assert torch.equal(got[side][b].nan_to_num(-9.25), self.model.values(side, b).nan_to_num(-9.25)), (side, b)
        self.cache.check()

    def attend(self, counts, heads, window=0, weight=None, **kw):
        q = torch.randn(sum(counts), heads, self.D, generator=self.g).to(self.dtype)
        one = all(n == 1 for n in counts)
        out, lse = self.cache.attend(q.to(self.device), self.table, self.lens(), None if one else self.cu(counts), None if one else max(counts),
                                     scale=self.D ** -0.5, window=window, want_lse=True, weight=weight, **kw)
        return q, out.cpu(), lse.cpu()

    def close(self, q, out, lse, counts, window=0):
        """Compares one attend with the definition; the weights' sums [seqs][H, len] and their bounds."""
        sums, at = [], 0
        for b, n in enumerate(counts):
            k, v = (self.model.values(s, b) for s in range(2))
            qb = q[at: at + n]
            o, l, w = ref.attend(qb, k, v, self.D ** -0.5, window)
            assert torch.equal(torch.isnan(out[at: at + n]), torch.isnan(o))
            fine = ~torch.isnan(o)
            err = (out[at: at + n].double() - o).abs()
            bound = ref.attend_bound(qb, k.nan_to_num(0), v.nan_to_num(0), self.D ** -0.5, self.dtype, o.nan_to_num(0))
            assert bool((err <= bound)[fine].all()), (b, float((err / bound)[fine].max()))
            lb = ref.score_bound(qb, k.nan_to_num(0), self.D ** -0.5)
            ok = torch.isfinite(l)
            assert torch.equal(lse[at: at + n][~ok].double().nan_to_num(5.0), l[~ok].nan_to_num(5.0))
            assert bool(((lse[at: at + n].double() - l).abs() <= lb)[ok].all())
            # a weight exp(s - lse) is off by the two scores' errors, relatively, and the sum's roundings
            sums.append((w, w * (2 * float(lb.max() if lb.numel() else 0) + (n * q.shape[1] // self.H + 8) * 2.0 ** -24)))
            at += n
        self.cache.check()
        return sums


# ---------------------------------------------------------------- rotary

@pytest.mark.parametrize("dtype", [F16, BF16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,heads,kv,dim,rot", [(1, 16, 8, 128, 128), (7, 3, 1, 128, 96), (33, 5, 5, 64, 26), (5, 2, 0, 256, 254), (3, 4, 2, 80, 2),
                                                (257, 9, 3, 128, 64), (2, 1, 1, 6, 6), (4, 3, 2, 256, 256)])
def test_rope(kv8, dtype, layout, T, heads, kv, dim, rot):
    g = torch.Generator().manual_seed(T + rot)
    freq, factor = kv8.rope_freqs(rot, 1e6, "yarn", 4.0)
    pos = torch.randint(-5, 1000000, (T,), generator=g, dtype=torch.int32)
    q, k = torch.randn(T, heads, dim, generator=g).to(dtype), torch.randn(T, kv, dim, generator=g).to(dtype)
    got = kv8.rope(q.cuda(), k.cuda() if kv else None, pos.cuda(), freq.cuda(), layout=layout, factor=factor)
    for x, y in ((q, got[0]), (k, got[1])):
        if y is None:
            continue
        want = ref.rope(x, pos, freq, layout, factor)
        # cos and sin: the reduced angle in float32 (2 pi * 2^-25 rad), their own two units, the factor; the product and the sum;
        # and the two ways of 64 bits of forming pos * freq (1e6 rad * 2^-52)
        mag = x.double().abs().amax(-1, keepdim=True) * 2 * factor
        tol = mag * (2 * math.pi * 2.0 ** -25 + 5 * 2.0 ** -24 + 1e-9) + torch.finfo(dtype).eps / 2 * want.abs()
        assert bool(((y.cpu().double() - want).abs() <= tol * 1.0001).all())
        assert torch.equal(y.cpu()[..., rot:], x[..., rot:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_in_place_on_strided_heads_and_unaligned_rows(kv8, layout):
    g = torch.Generator().manual_seed(3)
    freq, _ = kv8.rope_freqs(128, 1e4)
    pos = torch.arange(11, dtype=torch.int32)
    for pad in (0, 1, 3):                                  # a fused q | k | v buffer, rows at odd offsets
        buf = torch.randn(11, 6 * 128 + pad, generator=g).to(F16)
        dev = buf.cuda()
        view = lambda t, a, n: t[:, pad + a * 128: pad + (a + n) * 128].unflatten(1, (n, 128))  # noqa: E731
        q, k = view(dev, 0, 3), view(dev, 3, 2)
        kv8.rope(q, k, pos.cuda(), freq.cuda(), layout=layout, q_out=q, k_out=k)
        fresh = kv8.rope(view(buf.cuda(), 0, 3), view(buf.cuda(), 3, 2), pos.cuda(), freq.cuda(), layout=layout)
        assert torch.equal(q, fresh[0]) and torch.equal(k, fresh[1])
        assert torch.equal(dev[:, :pad].cpu(), buf[:, :pad]) and torch.equal(dev[:, pad + 640:].cpu(), buf[:, pad + 640:])
        want = ref.rope(view(buf, 0, 3), pos, freq, layout, 1.0)
        assert bool(((q.cpu().double() - want).abs() <= 2 * buf.abs().max() * 2.0 ** -21 + want.abs() * 2.0 ** -11).all())


def test_rope_of_nothing(kv8):
    freq, _ = kv8.rope_freqs(64, 1e4)
    q, k = kv8.rope(torch.zeros(0, 4, 64, dtype=F16, device="cuda"), None, torch.zeros(0, dtype=torch.int32, device="cuda"), freq.cuda())
    assert q.shape == (0, 4, 64) and k is None


# ---------------------------------------------------------------- append and read

@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,H", [(64, 3), (128, 2), (256, 1)])
def test_append_is_the_definition_however_rows_arrive(kv8, code, dtype, D, H):
    steps = [[5, 0, 33, 17], [1, 1, 1, 1], [10, 64, 0, 100], [1, 1, 1, 1], [0, 0, 15, 16], [15, 3, 16, 31], [1, 1, 1, 1], [40, 2, 1, 0]]
    a = Both(kv8, 4, H, D, code, dtype, cols=4, seed=D)
    for counts in steps:
        a.append(counts)
        a.same()
    # all at once: the same bits
    b = Both(kv8, 4, H, D, code, dtype, cols=4, seed=1)
    counts = [r.shape[0] for r in a.model.rows[0]]
    b.append(counts, *[torch.cat(a.model.rows[s]) for s in range(2)])
    for s in range(2):
        for x, y in zip(a.read()[s], b.read()[s]):
            assert torch.equal(x, y)


def test_append_takes_rows_back(kv8):
    a = Both(kv8, 2, 2, 128, "int8", F16, cols=3)
    a.append([47, 100])
    for back, n in [([16, 16], [3, 20]), ([1, 2], [1, 1]), ([14, 9], [40, 16])]:
        for b in range(2):
            a.model.cut(b, a.model.rows[0][b].shape[0] - back[b])
        a.append(n)
        a.same()


def test_append_leaves_other_pages_and_blocks_alone(kv8):
    a = Both(kv8, 2, 2, 64, "int8", F16, cols=3, spare=2)
    a.append([20, 0])
    c = a.cache
    used = a.table[0, 0].item()
    for t in (c.k, c.v):
        x = t.view(torch.uint8).cpu()
        assert bool((x[[i for i in range(8) if i != used]] == 255).all()) and bool((x[used, :, 32:] == 255).all())
        assert bool((x[used, :, 20:32] == 0).all())
    for t in (c.k_scale, c.v_scale):
        x = t.cpu()
        assert int(torch.isnan(x).sum()) == x.numel() - 4
    assert bool(torch.isnan(c.k_open[1]).all())


def test_append_of_values_at_the_edges(kv8):
    for dtype, code in ((F16, "int8"), (F16, "e4m3"), (BF16, "int8"), (BF16, "e4m3")):
        big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        x = torch.randn(16 * 6, 1, 64, generator=torch.Generator().manual_seed(9)).to(dtype)
        x[:16] = 0
        x[16:32] *= tiny * 40 if dtype is F16 else 0
        x[16, 0, 0] = tiny
        x[32, 0, 5] = big
        x[33, 0, 6] = -big
        x[48, 0, 1] = math.inf
        x[64, 0, 1] = -math.inf
        x[80, 0, 63] = math.nan
        a = Both(kv8, 1, 1, 64, code, dtype, cols=2)
        a.append([96], x, x.flip(0).contiguous())
        a.same()
        k, v = a.read()
        assert bool(torch.isnan(k[0][48:]).all()) and bool(torch.isfinite(k[0][:48]).all()) and bool(torch.isnan(v[0][:48]).all())


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append_rounds_every_quotient_correctly(kv8, code, dtype):
    """Every mantissa of a block's largest magnitude against every value of the eleven binades below it (F16; all of BF16's
    mantissas twice over): ties are exact quotients, so one wrong bit of a quotient shows."""
    bits = 10 if dtype is F16 else 7
    m = torch.arange(2 ** bits, dtype=torch.float64) / 2 ** bits + 1
    below = torch.cat([m * 2.0 ** -e for e in range(11)])                       # 11 * 2^bits values up to 2
    per = 11 if dtype is F16 else 2
    x = torch.zeros(2 ** bits, per, 1024, dtype=torch.float64)
    v = below.repeat(2)[: per * 1023].reshape(per, 1023)
    x[:, :, 1:] = torch.minimum(v[None], m[:, None, None])
    x[:, :, 0] = m[:, None]
    x[:, :, 2::3] *= -1
    x = x.reshape(-1, 1, 64).to(dtype)
    n = x.shape[0]
    a = Both(kv8, 1, 1, 64, code, dtype, cols=-(-n // 64))
    a.append([n], x, x.flip(0).contiguous())
    a.same()


@pytest.mark.parametrize("pad", [0, 1, 8])
def test_append_of_strided_rows(kv8, pad):
    a = Both(kv8, 3, 2, 128, "int8", BF16, cols=2)
    n = [33, 5, 64]
    buf = rows(a.g, sum(n), 6, 128, BF16).flatten(1)
    buf = torch.cat([torch.zeros(sum(n), pad, dtype=BF16), buf], 1).cuda()
    view = buf[:, pad:].unflatten(1, (6, 128))
    k, v = view[:, 2:4], view[:, 4:6]
    at = 0
    for b, m in enumerate(n):
        a.model.append(b, k[at: at + m].cpu(), v[at: at + m].cpu())
        at += m
    a.cache.append(k, v, a.table, a.lens(), a.cu(n), 64)
    a.same()


@pytest.mark.parametrize("dtype", [F16, BF16, torch.float32])
def test_read_of_a_part(kv8, dtype):
    a = Both(kv8, 3, 2, 128, "e4m3", F16, cols=3)
    a.append([150, 0, 64])
    begin, n = [100, 0, 63], [50, 0, 1]
    k, v = a.cache.read(a.table, torch.tensor(begin, dtype=torch.int32, device="cuda"), a.cu(n), 51, 50, dtype)
    for side, x in ((0, k), (1, v)):
        want = torch.cat([a.model.values(side, b)[i: i + m] for b, (i, m) in enumerate(zip(begin, n))]).to(dtype)
        assert torch.equal(x.cpu(), want)
    a.cache.check()


# ---------------------------------------------------------------- attention

LENS = [1, 15, 16, 17, 63, 64, 65, 130, 300]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,H,heads", [(128, 2, 4), (64, 1, 5), (256, 1, 2), (128, 1, 16), (128, 3, 3), (64, 2, 22), (128, 1, 40), (256, 1, 17)])
def test_attend_one_row_each(kv8, code, dtype, D, H, heads):
    a = Both(kv8, len(LENS), H, D, code, dtype, cols=5, seed=heads)
    a.append(LENS)
    n = [1] * len(LENS)
    a.close(*a.attend(n, heads), n)


@pytest.mark.parametrize("window", [1, 16, 50])
def test_attend_windows(kv8, window):
    a = Both(kv8, len(LENS), 2, 128, "int8", F16, cols=5)
    a.append(LENS)
    n = [1] * len(LENS)
    a.close(*a.attend(n, 4, window), n, window)
    n = [1, 9, 16, 2, 0, 40, 65, 100, 3]
    a.close(*a.attend(n, 4, window), n, window)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,H,heads,n", [(128, 2, 4, [1, 15, 7, 17, 0, 64, 3, 130, 90]), (64, 1, 5, [1, 1, 2, 3, 4, 3, 2, 1, 3]),
                                         (128, 1, 8, [1, 2, 2, 2, 2, 2, 2, 2, 2]), (256, 1, 2, [1, 15, 16, 17, 63, 64, 65, 1, 299]),
                                         (64, 2, 6, [0, 0, 0, 0, 0, 0, 0, 130, 257]),
                                         (64, 8, 16, [1, 15, 16, 17, 20, 20, 0, 3, 20]), (128, 8, 32, [0, 9, 10, 11, 12, 1, 16, 16, 15])])
def test_attend_several_rows(kv8, code, dtype, D, H, heads, n):
    a = Both(kv8, len(LENS), H, D, code, dtype, cols=5, seed=7)
    a.append(LENS)
    a.close(*a.attend(n, heads), n)


@pytest.mark.parametrize("n", [[1, 1, 1], [4, 0, 9], [100, 2, 90]])
def test_rows_that_see_nothing(kv8, n):
    # an empty sequence; and rows before the first position (more rows than the sequence is long)
    a = Both(kv8, 3, 2, 128, "int8", F16, cols=2)
    a.append([2, 0, 70])
    q, out, lse = a.attend(n, 4)
    a.close(q, out, lse, n)
    assert bool(torch.isneginf(lse).any()) and bool((out[torch.isneginf(lse)] == 0).all())


def test_long_and_ragged(kv8):
    lens = [9000, 1, 0, 2500, 33]
    a = Both(kv8, 5, 2, 128, "int8", F16, cols=141)
    a.append(lens)
    for n, heads, window in [([1] * 5, 4, 0), ([1] * 5, 16, 4097), ([7, 1, 1, 0, 20], 4, 0), ([300, 1, 0, 129, 33], 4, 0)]:
        a.close(*a.attend(n, heads, window), n, window)


def test_one_long_sequence_split_over_the_gpu(kv8):
    a = Both(kv8, 1, 1, 128, "e4m3", BF16, cols=320)
    a.append([20471])
    for heads in (1, 6):
        a.close(*a.attend([1], heads), [1])


def test_hostile_values_in_places_that_no_row_sees(kv8):
    """NaN and infinities in blocks outside the window, and in the pages' unused rows (which Both fills), change nothing;
    a block of NaN that is seen gives NaN for exactly the rows that see it."""
    a = Both(kv8, 2, 1, 64, "e4m3", F16, cols=4)
    k = rows(a.g, 256 + 40, 1, 64, F16)
    v = k.flip(0).contiguous()
    k[3, 0, 3], v[20, 0, 1], v[70, 0, 60] = math.nan, math.inf, math.nan
    a.append([256, 40], k, v)
    n = [100, 40]
    a.close(*a.attend(n, 3, 64), n, 64)
    n = [1, 1]
    q, out, lse = a.attend(n, 3, 20)
    a.close(q, out, lse, n, 20)
    assert bool(torch.isfinite(out[0]).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_large_and_small_values(kv8, dtype):
    a = Both(kv8, 2, 1, 128, "int8", dtype, cols=2)
    k, v = rows(a.g, 100, 1, 128, dtype), rows(a.g, 100, 1, 128, dtype)
    v[:40] *= torch.tensor(1e-4).to(dtype)
    v[40:60] *= torch.tensor(500.0).to(dtype)
    a.append([60, 40], k, v)
    # scores far apart: one key takes all
    q = (torch.randn(2, 4, 128, generator=a.g) * 60).to(dtype)
    out, lse = a.cache.attend(q.cuda(), a.table, a.lens(), scale=128 ** -0.5, want_lse=True)
    a.close(q, out.cpu(), lse.cpu(), [1, 1])
    # queries below F16's smallest normal number
    q = (torch.randn(2, 4, 128, generator=a.g) * 1e-6).to(dtype)
    out, lse = a.cache.attend(q.cuda(), a.table, a.lens(), scale=1000.0, want_lse=True)
    for b in range(2):
        o, l, _ = ref.attend(q[b: b + 1], a.model.values(0, b), a.model.values(1, b), 1000.0)
        bound = ref.attend_bound(q[b: b + 1], a.model.values(0, b), a.model.values(1, b), 1000.0, dtype, o)
        assert bool(((out[b: b + 1].cpu().double() - o).abs() <= bound).all())


def test_attend_of_strided_queries_into_strided_rows_leaves_the_rest(kv8):
    a = Both(kv8, 3, 2, 64, "int8", F16, cols=2)
    a.append([70, 5, 128])
    n = [3, 0, 20]
    for pad in (0, 1, 8):
        big = torch.randn(30, 7 * 64 + pad, generator=a.g).to(F16).cuda()
        q = big[:, pad:].unflatten(1, (7, 64))[:, 1:5]
        o = torch.full((30, 9 * 64 + pad), 7.0, dtype=F16, device="cuda")
        out = o[:, pad:].unflatten(1, (9, 64))[:, 3:7]
        a.cache.attend(q, a.table, a.lens(), a.cu(n), 20, scale=64 ** -0.5, out=out)
        flat, _ = a.cache.attend(q[:23].contiguous(), a.table, a.lens(), a.cu(n), 20, scale=64 ** -0.5)
        assert torch.equal(out[:23], flat)
        keep = torch.ones_like(o, dtype=torch.bool)
        keep[:, pad:].unflatten(1, (9, 64))[:23, 3:7] = False
        assert bool((o[keep] == 7.0).all())


# ---------------------------------------------------------------- weights

@pytest.mark.parametrize("D,H,heads,n,window", [(128, 2, 4, [1, 1, 1, 1], 0), (64, 1, 5, [1, 1, 1, 1], 40), (128, 1, 8, [3, 0, 9, 1], 0),
                                                (256, 1, 3, [1, 16, 200, 10], 0), (128, 2, 2, [100, 40, 300, 15], 70), (64, 2, 40, [1, 1, 1, 1], 0)])
@pytest.mark.parametrize("code,dtype", [("int8", F16), ("e4m3", BF16)])
def test_weights(kv8, D, H, heads, n, window, code, dtype):
    a = Both(kv8, 4, H, D, code, dtype, cols=5)
    a.append([200, 40, 300, 15])
    start = torch.rand(4, H, 320 + 7, generator=a.g)
    w, wo = start.cuda(), torch.full((4, H, 320 + 7), -3.0, device="cuda")
    q, out, lse = a.attend(n, heads, window, weight=w, weight_out=wo)
    sums = a.close(q, out, lse, n, window)
    assert torch.equal(w.cpu(), start)
    for b, (s, bound) in enumerate(sums):
        L = s.shape[1]
        got = wo[b].cpu()
        want = start[b, :, :L].double() + s
        assert bool(((got[:, :L].double() - want).abs() <= bound + want.abs() * 2.0 ** -23).all())
        assert bool((got[:, L:] == -3.0).all())
    # in place, and the same sums
    q2, out2 = q.cuda(), torch.empty_like(out, device="cuda")
    one = all(m == 1 for m in n)
    a.cache.attend(q2, a.table, a.lens(), None if one else a.cu(n), None if one else max(n), scale=D ** -0.5, window=window, weight=w, out=out2)
    assert torch.equal(out2.cpu(), out)
    for b, (s, _) in enumerate(sums):
        assert torch.equal(w[b, :, :s.shape[1]], wo[b, :, :s.shape[1]])
        assert torch.equal(w[b, :, s.shape[1]:].cpu(), start[b, :, s.shape[1]:])


# ---------------------------------------------------------------- eviction

def _evict(a, weight, budget, sinks, recent):
    cols = -(-budget // 64)
    dst = a.spare[: a.seqs * cols].reshape(a.seqs, cols).contiguous()
    lens, keep, w = a.cache.evict(a.table, a.lens(), dst, weight.cuda(), budget, sinks=sinks, recent=recent)
    got = []
    counts = lens.tolist()
    k, v = a.cache.read(dst, None, a.cu(counts), sum(counts), max(counts), torch.float32)
    for b in range(a.seqs):
        n = a.model.rows[0][b].shape[0]
        assert counts[b] == min(n, budget)
        for h in range(a.H):
            at = ref.keep(weight[b, h], n, budget, sinks, recent)
            assert keep[b, h].tolist() == at + [-1] * (budget - len(at)), (b, h)
            assert torch.equal(w[b, h].cpu().nan_to_num(-2.0), torch.cat([weight[b, h][at], torch.zeros(budget - len(at))]).nan_to_num(-2.0))
            got.append((b, h, at))
    a.cache.check()
    k, v = k.cpu().split(counts), v.cpu().split(counts)
    for b, h, at in got:
        for side, x in ((0, k), (1, v)):
            code, scale = a.model.blocks(side, b)
            if not at:
                continue
            c = code.float().transpose(1, 2).reshape(-1, a.H, a.D)[at, h]
            s = scale.repeat_interleave(16, 0)[at, h]
            pad = -len(at) % 16
            nc, ns = ref.requantise(torch.cat([c, torch.zeros(pad, a.D)]), torch.cat([s, torch.zeros(pad)]), a.code)
            want = (nc.float() * ns[:, None, None]).reshape(-1, a.D)[: len(at)]
            assert torch.equal(x[b][:, h].nan_to_num(-2.0), want.nan_to_num(-2.0)), (b, h, side)
    return lens, keep, w, dst


@pytest.mark.parametrize("code,dtype,D,H", [("int8", F16, 128, 2), ("e4m3", BF16, 64, 3), ("int8", BF16, 256, 1), ("e4m3", F16, 128, 1)])
@pytest.mark.parametrize("budget,sinks,recent", [(16, 0, 0), (64, 4, 20), (96, 0, 96), (96, 96, 0), (80, 40, 40), (320, 3, 100), (48, 0, 1)])
def test_evict(kv8, code, dtype, D, H, budget, sinks, recent):
    lens = [300, 0, 64, 65, 17, 97]
    a = Both(kv8, 6, H, D, code, dtype, cols=5, spare=6 * 5, seed=budget)
    a.append(lens)
    _evict(a, torch.rand(6, H, 320, generator=a.g) ** 3, budget, sinks, recent)


def test_evict_with_ties_nan_and_odd_weights(kv8):
    a = Both(kv8, 4, 1, 64, "int8", F16, cols=40, spare=40)
    a.append([2500, 2500, 2048, 100])
    w = torch.zeros(4, 1, 2560)
    w[0] = torch.randint(0, 3, (1, 2560), generator=a.g).float()
    w[1, 0, ::7] = math.nan
    w[1, 0, 3::5] = -1.0
    w[1, 0, 4::5] = -0.0
    w[1, 0, 5::35] = math.inf
    w[2] = torch.rand(1, 2560, generator=a.g) * 1e-38
    _evict(a, w, 512, 5, 77)


def test_evict_flags_a_destination_in_use(kv8):
    a = Both(kv8, 1, 1, 64, "int8", F16, cols=4, spare=1)
    a.append([200])
    a.cache.evict(a.table, a.lens(), a.table[:, 3:4].contiguous(), torch.rand(1, 1, 256, device="cuda"), 64)
    with pytest.raises(RuntimeError, match="in use"):
        a.cache.check()


def test_evict_keeps_blocks_that_move_whole(kv8):
    a = Both(kv8, 1, 2, 128, "e4m3", BF16, cols=4, spare=4)
    a.append([256])
    w = torch.zeros(1, 2, 256)
    w[0, 0, 32:64], w[0, 1, 96:128] = 1.0, 1.0
    _, keep, _, dst = _evict(a, w, 64, 16, 16)
    old, new = a.read()[0][0], a.cache.read(dst, None, a.cu([64]), 64, 64, torch.float32)[0].cpu()
    for h in range(2):
        assert torch.equal(new[:, h], old[keep[0, h].tolist(), h])


# ---------------------------------------------------------------- device-side checks, streams, graphs, the loop

def test_bad_pages_and_lengths_are_left_out(kv8):
    """Run after the same bounds passed on the CPU (tests/test_kv8_cpu.py): a page number outside the pool hides its keys."""
    a = Both(kv8, 2, 1, 64, "int8", F16, cols=3)
    a.append([150, 64])
    good, lens = a.table.clone(), a.lens()
    q = torch.randn(2, 2, 64, generator=a.g).to(F16)
    for bad in (6, -1, 2 ** 31 - 1, -2 ** 31):
        a.table = good.clone()
        a.table[0, 1] = bad
        for w in (None, torch.zeros(2, 1, 192, device="cuda")):
            out, _ = a.cache.attend(q.cuda(), a.table, lens, scale=0.125, weight=w)
            with pytest.raises(RuntimeError, match="page"):
                a.cache.check()
            k, v = (a.model.values(s, 0) for s in range(2))
            part = [torch.cat([x[:64], x[128:]]) for x in (k, v)]
            o, _, _ = ref.attend(q[:1], *part, 0.125)
            assert bool(((out[:1].cpu().double() - o).abs() <= ref.attend_bound(q[:1], *part, 0.125, F16, o)).all())
        a.cache.append(q[:, :1].contiguous().cuda(), q[:, :1].contiguous().cuda(), a.table, torch.tensor([100, 64], dtype=torch.int32, device="cuda"))
        with pytest.raises(RuntimeError, match="page"):
            a.cache.check()
        a.cache.read(a.table, None, a.cu([150, 64]), 214, 150)
        with pytest.raises(RuntimeError, match="page"):
            a.cache.check()
        a.cache.evict(a.table, lens, torch.full((2, 1), bad, dtype=torch.int32, device="cuda"), torch.rand(2, 1, 192, device="cuda"), 64)
        with pytest.raises(RuntimeError, match="page"):
            a.cache.check()
    a.table = good
    for n in (-1, 193, 2 ** 31 - 1):
        bad_lens = torch.tensor([n, 64], dtype=torch.int32, device="cuda")
        out = torch.full((2, 2, 64), 5.0, dtype=F16, device="cuda")
        a.cache.attend(q.cuda(), a.table, bad_lens, scale=0.125, out=out)
        with pytest.raises(RuntimeError, match="length"):
            a.cache.check()
        assert bool((out[0] == 5.0).all()) and not bool((out[1] == 5.0).any())
    for cu in ([0, 3, 2], [0, 1, 3], [-1, 1, 2], [0, 2, 2]):
        out = torch.full((2, 2, 64), 5.0, dtype=F16, device="cuda")
        a.cache.attend(q.cuda(), a.table, lens, torch.tensor(cu, dtype=torch.int32, device="cuda"), 1, scale=0.125, out=out)
        with pytest.raises(RuntimeError, match="rows"):
            a.cache.check()


def test_refusals(kv8):
    c = kv8.KvCache8.empty(4, 2, 2, 128)
    t, n = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    x = torch.zeros(2, 2, 128, dtype=F16, device="cuda")
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    f = torch.ones(64, dtype=torch.float64, device="cuda")
    w = torch.zeros(2, 2, 128, device="cuda")
    for call in [
        lambda: c.append(x.to(BF16), x.to(BF16), t, n), lambda: c.append(x[:1], x[:1], t, n), lambda: c.append(x, x[:, :1], t, n),
        lambda: c.append(x.cpu(), x, t, n), lambda: c.append(x, x, t.long(), n), lambda: c.append(x, x, t[:1], n), lambda: c.append(x, x, t, n[:1]),
        lambda: c.append(x, x, t, n.cpu()), lambda: c.append(x, x, t, n, cu), lambda: c.append(x, x, t, n, cu[:2], 1), lambda: c.append(x, x, t, n, cu, -1),
        lambda: c.append(x.transpose(1, 2), x.transpose(1, 2), t, n), lambda: c.append(x, x, t.t(), n), lambda: c.append(x, x, t[:, :0].contiguous(), n),
        lambda: c.read(t, None, cu, 2, 1, torch.float64), lambda: c.read(t, n.long(), cu, 2, 1), lambda: c.read(t, None, cu, -1, 1), lambda: c.read(t, None, None, 3, 1),
        lambda: c.attend(x[:, :1], t, n, scale=1.0), lambda: c.attend(x, t, n, cu, scale=1.0), lambda: c.attend(x, t, n, scale=1.0, window=-1), lambda: c.attend(x, t, n, scale=1.0, window=2 ** 40), lambda: c.attend(x, t, n, scale=-1.0),
        lambda: c.attend(x, t, n, cu, 2 ** 31 - 1, scale=1.0),
        lambda: c.attend(x, t, n, scale=1.0, weight=w[..., :127].contiguous()), lambda: c.attend(x, t, n, scale=1.0, weight_out=w),
        lambda: c.attend(x, t, n, scale=1.0, weight=w.half()), lambda: c.attend(x, t, n, scale=1.0, out=x[:1]), lambda: c.attend(x[:, :0], t, n, scale=1.0),
        lambda: c.evict(t, n, t.clone(), w, 24), lambda: c.evict(t, n, t.clone(), w, 0), lambda: c.evict(t, n, t.clone(), w, 144), lambda: c.evict(t, n, t, w, 16),
        lambda: c.evict(t, n, t.clone(), w, 16, sinks=10, recent=7), lambda: c.evict(t, n, t.clone(), w, 16, sinks=-1), lambda: c.evict(t, n, t.clone(), w[..., :64], 16),
        lambda: kv8.rope(x, x, n.long(), f), lambda: kv8.rope(x, x, n, f.float()), lambda: kv8.rope(x, x, n, f, layout="pairs"), lambda: kv8.rope(x, x[:1], n, f),
        lambda: kv8.rope(x, x, n, torch.ones(65, dtype=torch.float64, device="cuda")), lambda: kv8.rope(x, x, n, f[:0]), lambda: kv8.rope(x, x, n, f, q_out=x[:, :1]),
        lambda: kv8.rope(x, x, n, f, q_out=x.transpose(0, 1)), lambda: kv8.rope(x.int(), None, n, f), lambda: kv8.KvCache8.empty(4, 2, 2, 96),
        lambda: kv8.KvCache8(c.k, c.v, c.k_scale.half(), c.v_scale, c.k_open, c.v_open), lambda: kv8.KvCache8(c.k, c.v[:2], c.k_scale, c.v_scale, c.k_open, c.v_open),
        lambda: kv8.KvCache8(c.k.cpu(), c.v, c.k_scale, c.v_scale, c.k_open, c.v_open),
    ]:
        with pytest.raises(ValueError):
            call()
    c.check()


def _loop(kv8, a, q_heads, steps, freq, budget, graph=False):
    """Rotary, append, attend with weights, evict: `steps` tokens per sequence; outputs of every step."""
    H, D, B = a.H, a.D, a.seqs
    g = torch.Generator().manual_seed(5)
    xs = torch.randn(steps, B, q_heads + 2 * H, D, generator=g).to(a.dtype).cuda()
    x = xs[0].clone()
    lens = a.lens()
    pos = lens.clone()
    weight = torch.zeros(B, H, a.cols * 64, device="cuda")
    out = torch.empty(B, q_heads, D, dtype=a.dtype, device="cuda")

    def step():
        q, k = kv8.rope(x[:, :q_heads], x[:, q_heads: q_heads + H], pos, freq)
        lens.add_(1)
        pos.add_(1)
        a.cache.append(k, x[:, q_heads + H:], a.table, lens)
        a.cache.attend(q, a.table, lens, scale=D ** -0.5, weight=weight, out=out)

    outs = []
    if graph:
        keep = [t.clone() for t in (lens, pos, a.cache.k_open, a.cache.v_open)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        G = torch.cuda.CUDAGraph()
        with torch.cuda.graph(G):
            step()
        torch.cuda.synchronize()
        for t, s in zip((lens, pos, a.cache.k_open, a.cache.v_open), keep):
            t.copy_(s)
        weight.zero_()
    for i in range(steps):
        x.copy_(xs[i])
        G.replay() if graph else step()
        outs.append(out.clone())
    cols = -(-budget // 64)
    dst = a.spare[: B * cols].reshape(B, cols).contiguous()
    lens2, keep, w2 = a.cache.evict(a.table, lens, dst, weight, budget, sinks=2, recent=16)
    o, _ = a.cache.attend(xs[0][:, :q_heads].contiguous(), dst, lens2, scale=D ** -0.5)
    torch.cuda.synchronize()
    a.cache.check()
    return torch.stack(outs).cpu(), weight.cpu(), keep.cpu(), o.cpu(), xs.cpu(), lens2.cpu()


def test_a_decode_loop(kv8):
    """The operators together, as a serving loop runs them, against the same loop in float64 (with the cache's own rounding of k and v);
    then the same loop replayed from a captured graph, and on another stream: the same bits."""
    B, H, heads, D, steps, budget = 3, 2, 4, 128, 40, 64
    freq, _ = kv8.rope_freqs(D, 1e6)
    make = lambda: Both(kv8, B, H, D, "int8", F16, cols=4, spare=2 * B, seed=11)  # noqa: E731
    a = make()
    a.append([70, 0, 150])
    outs, weight, keep, o, xs, lens = _loop(kv8, a, heads, steps, freq.cuda(), budget)
    total = [torch.zeros(H, 256, dtype=torch.float64) for _ in range(B)]
    pos = [70, 0, 150]
    for i in range(steps):
        for b in range(B):
            p = torch.tensor([pos[b]], dtype=torch.int32)
            # the rotated heads as the operator gives them (tested above): one rounding of the exact values may differ
            q, k = kv8.rope(xs[i][b: b + 1, :heads].cuda(), xs[i][b: b + 1, heads: heads + H].cuda(), p.cuda(), freq.cuda())
            a.model.append(b, k.cpu(), xs[i][b: b + 1, heads + H:])
            pos[b] += 1
            kk, vv = (a.model.values(s, b) for s in range(2))
            ref_o, _, w = ref.attend(q.cpu(), kk, vv, D ** -0.5)
            assert bool(((outs[i, b: b + 1].double() - ref_o).abs() <= ref.attend_bound(q.cpu(), kk, vv, D ** -0.5, F16, ref_o)).all())
            total[b][:, : w.shape[1]] += w
    for b in range(B):
        assert float((weight[b].double() - total[b]).abs().max()) < 1e-4 * heads / H
        for h in range(H):
            at = ref.keep(weight[b, h], pos[b], budget, 2, 16)
            assert keep[b, h].tolist() == at + [-1] * (budget - len(at))
    assert lens.tolist() == [64, 40, 64] and bool(torch.isfinite(o).all())
    a.same()

    b = make()
    b.append([70, 0, 150])
    again = _loop(kv8, b, heads, steps, freq.cuda(), budget, graph=True)
    c = make()
    with torch.cuda.stream(torch.cuda.Stream()):
        c.append([70, 0, 150])
        other = _loop(kv8, c, heads, steps, freq.cuda(), budget)
    for x, y, z in zip((outs, weight, keep, o), again, other):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_calls_on_two_streams_at_once(kv8):
    """Two caches, two streams, interleaved calls: the bits of one after the other."""
    n, heads = [1] * 4, 8
    caches = []
    for s in range(2):
        a = Both(kv8, 4, 2, 128, "int8", F16, cols=70, seed=s)
        a.append([4000, 100, 3000, 4480])
        caches.append(a)
    qs = [torch.randn(4, heads, 128, generator=a.g).to(F16).cuda() for a in caches]
    alone = [a.cache.attend(q, a.table, a.lens(), scale=0.1)[0] for a, q in zip(caches, qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    lens = [a.lens() for a in caches]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, a in enumerate(caches):
            with torch.cuda.stream(streams[i]):
                got[i].append(a.cache.attend(qs[i], a.table, lens[i], scale=0.1)[0])
    torch.cuda.synchronize()
    for i in range(2):
        for x in got[i]:
            assert torch.equal(x, alone[i])


def test_offsets_past_32_bits(kv8):
    """A pool of more than 2^32 codes: the last pages are read and written where they are."""
    pages, H, D = 66000, 8, 128                       # 66000 * 8 * 64 * 128 = 4.3e9 codes a side
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    c = kv8.KvCache8.empty(pages, 1, H, D)
    g = torch.Generator().manual_seed(1)
    k, v = rows(g, 100, H, D, F16), rows(g, 100, H, D, F16)
    lens = torch.tensor([100], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 100], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 16, D, generator=g).to(F16).cuda()
    got = []
    for table in ([65999, 65535], [0, 1]):
        t = torch.tensor([table], dtype=torch.int32, device="cuda")
        c.append(k.cuda(), v.cuda(), t, lens, cu, 100)
        got.append((c.attend(q, t, lens, scale=0.1)[0], *c.read(t, None, cu, 100, 100)))
    for x, y in zip(*got):
        assert torch.equal(x, y)
    c.check()


def test_the_callers_device_stays(kv8):
    L = kv8._lib()
    a = kv8.RopeArgs(99, 1, 1, 1, 0, 64, 64, 0, 1.0, 4096, 4096, 4096, None, 8192, None)
    assert L.qtts_op_rope(C.byref(a), None) == 0 and "device" in L.qtts_create_error().decode()
    assert torch.cuda.current_device() == 0
    torch.zeros(1, device="cuda").add_(1)
    torch.cuda.synchronize()
