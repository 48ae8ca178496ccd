"""The decode loop's operators around the 8-bit key/value cache: rotary positions, append, attention, eviction.

Every case names an operator, its sizes and the ragged lengths that it draws from `ragged`; the values come from the seed.
The cache is a pool of pages of 64 tokens. A page holds, for each key/value head, 64 rows of 8-bit codes (int8, or 8-bit floats with 4 exponent
bits) for the keys and for the values, and one 32-bit scale for each block of 16 tokens. The rows of a sequence's last two blocks are also kept in
16 bits, in a ring of 32 rows for each sequence and head, so that a block that is still filling up is quantised from its 16-bit rows.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

PAGE, BLOCK, RING = 64, 16, 32
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
TOP = {"int8": 127.0, "e4m3": 448.0}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one sequence's query and key heads on their way into a step, the talker's own layout
        dict(name="rope, one token", op="rope", rows=1, heads=16, kv_heads=8, dim=128, rot=128, layout="half", scaling="none", factor=1.0, theta=1e6,
             type="f16", far=4500),
        # a long prompt of another layout: interleaved pairs on three quarters of the head, positions stretched eight times
        dict(name="rope, long prompt, interleaved, scaled", op="rope", rows=16411, heads=32, kv_heads=4, dim=128, rot=96, layout="interleaved",
             scaling="yarn", factor=8.0, theta=1e4, type="bf16", far=250000),
        # one frame of 32 long utterances: a row for each of them
        dict(name="append, a step of 32", op="append", seqs=32, heads=16, kv_heads=8, dim=128, code="int8", type="f16", len_min=3900, len_max=4608,
             new_min=1, new_max=1, ragged=1),
        # 64 prompts of 32 to 512 positions, as a batch begins
        dict(name="append, 64 prompts", op="append", seqs=64, heads=16, kv_heads=8, dim=128, code="e4m3", type="bf16", len_min=32, len_max=512,
             new_min=0, new_max=0, ragged=2),
        # the first frames of one utterance: latency is all that counts
        dict(name="attend, one short sequence", op="attend", seqs=1, heads=16, kv_heads=8, dim=128, code="int8", type="f16", len_min=197, len_max=197,
             q_min=1, q_max=1, window=0, ragged=3, weigh=False, lse=False),
        # a frame of the long-form batch: 32 utterances at some 4,400 positions
        dict(name="attend, a step of 32 at 4400", op="attend", seqs=32, heads=16, kv_heads=8, dim=128, code="int8", type="f16", len_min=4200, len_max=4608,
             q_min=1, q_max=1, window=0, ragged=4, weigh=False, lse=False),
        # two very long contexts and few heads: work has to be split along the cache
        dict(name="attend, a step at 131072", op="attend", seqs=2, heads=32, kv_heads=4, dim=128, code="e4m3", type="bf16", len_min=120001, len_max=131072,
             q_min=1, q_max=1, window=0, ragged=5, weigh=False, lse=True),
        # chunks of several prompts over what is cached of them
        dict(name="attend, chunks of 8 prompts", op="attend", seqs=8, heads=16, kv_heads=8, dim=128, code="int8", type="f16", len_min=700, len_max=2100,
             q_min=100, q_max=512, window=0, ragged=6, weigh=False, lse=True),
        # a long chunk of one long prompt
        dict(name="attend, a chunk of 2048 at 16384", op="attend", seqs=1, heads=32, kv_heads=4, dim=128, code="int8", type="bf16", len_min=16384, len_max=16384,
             q_min=2048, q_max=2048, window=0, ragged=7, weigh=False, lse=False),
        # a step that also adds up what each cached token was attended with, in a model of 64-wide heads in groups of five
        dict(name="attend, a weighing step of 16", op="attend", seqs=16, heads=40, kv_heads=8, dim=64, code="int8", type="f16", len_min=1500, len_max=2500,
             q_min=1, q_max=1, window=0, ragged=8, weigh=True, lse=True),
        # four caches that have grown past their budget by a little
        dict(name="evict, 4 down to 512", op="evict", seqs=4, heads=16, kv_heads=8, dim=128, code="int8", type="f16", len_min=400, len_max=768, budget=512,
             sinks=4, recent=128, ragged=9),
        # eight long contexts cut to a quarter
        dict(name="evict, 8 from 32768 to 8192", op="evict", seqs=8, heads=16, kv_heads=8, dim=128, code="e4m3", type="bf16", len_min=30000, len_max=32768,
             budget=8192, sinks=16, recent=1024, ragged=10),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "append", "step", "chunk", "weigh", "evict"])
    group = rng.choice([1, 2, 3, 4, 5, 8, 16])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 128, 128, 256])
    base = dict(heads=group * kv_heads, kv_heads=kv_heads, dim=dim, type=rng.choice(["f16", "bf16"]))
    if kind == "rope":
        far = _log(rng, 100, 1000000)
        return dict(base, op="rope", rows=_log(rng, 1, min(32768, 2 ** 26 // ((group + 1) * kv_heads * dim))), rot=2 * rng.randint(4, dim // 2), layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "ntk", "yarn"]), factor=float(rng.choice([2, 4, 8, 32])), theta=rng.choice([1e4, 5e5, 1e6]),
                    far=far)
    base.update(code=rng.choice(["int8", "e4m3"]), ragged=rng.randint(11, 10 ** 6))
    if kind == "append":
        if rng.random() < 0.5:
            n = rng.randint(1, 8)
            hi = _log(rng, 64, 8192)
            return dict(base, op="append", seqs=_log(rng, 1, 64), len_min=hi // 2, len_max=hi, new_min=rng.randint(0, n), new_max=n)
        hi = _log(rng, 8, 4096)
        return dict(base, op="append", seqs=_log(rng, 1, max(1, 2 ** 22 // (hi * dim))), len_min=rng.randint(0, hi), len_max=hi, new_min=0, new_max=0)
    if kind == "chunk":
        hi = _log(rng, 20, 8192)
        q = _log(rng, 2, max(2, min(hi, 1024, 10 ** 11 // (hi * group * kv_heads * dim))))
        return dict(base, op="attend", seqs=max(1, min(16, 2 ** 24 // (hi * q * group * kv_heads // 8 + 1))), len_min=rng.randint(q, hi), len_max=hi,
                    q_min=rng.randint(1, q), q_max=q, window=rng.choice([0, 0, 0, rng.randint(1, hi)]), weigh=rng.random() < 0.25,
                    lse=rng.random() < 0.5)
    hi = _log(rng, 3, 65536)
    seqs = _log(rng, 1, max(1, min(64, 2 ** 27 // (hi * kv_heads * dim))))
    if kind == "evict":
        hi = max(hi, 100)
        budget = 16 * _log(rng, 2, max(2, hi // 16))
        sinks = rng.randint(0, min(32, budget // 4))
        return dict(base, op="evict", seqs=min(seqs, max(1, 2 ** 26 // (hi * kv_heads * dim))), len_min=rng.randint(0, hi), len_max=hi, budget=budget, sinks=sinks,
                    recent=rng.randint(0, budget - sinks))
    return dict(base, op="attend", seqs=seqs, len_min=rng.randint(0, hi), len_max=hi, q_min=1, q_max=1, window=rng.choice([0, 0, 0, rng.randint(1, hi)]),
                weigh=kind == "weigh", lse=rng.random() < 0.5)


def _lengths(case):
    """Each sequence's length, and how many of its last rows the call brings (new rows, or queries)."""
    r = random.Random(case["ragged"])
    lens = [r.randint(case["len_min"], case["len_max"]) for _ in range(case["seqs"])]
    lens[r.randrange(len(lens))] = case["len_max"]
    if case["op"] == "append":
        new = [min(n, r.randint(case["new_min"], case["new_max"])) if case["new_max"] else n for n in lens]
    elif case["op"] == "attend":
        new = [min(n, r.randint(case["q_min"], case["q_max"])) if case["q_max"] > 1 else 1 for n in lens]
    else:
        new = [min(n, case["budget"]) for n in lens]
    return lens, new


# ---------------------------------------------------------------- inputs

def _frequencies(case):
    """Angle per position of each pair, in 64 bits, and the factor on the rotated values (a program keeps both for its model)."""
    i = torch.arange(0, case["rot"], 2, dtype=torch.float64)
    theta, factor, rot = case["theta"], case["factor"], case["rot"]
    if case["scaling"] == "ntk" and rot > 2:
        theta = theta * factor ** (rot / (rot - 2))
    f = theta ** (-i / rot)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "yarn":
        at = [rot * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(theta)) for turns in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        ramp = ((torch.arange(rot // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _rows(shape, dtype, g):
    """Key or value rows as projections leave them: some channels of each head are several times as large as the rest."""
    size = 0.5 + torch.rand(shape[-1], device="cuda", generator=g)
    size[:: 16] *= 6
    return (torch.randn(shape, device="cuda", generator=g) * size).to(dtype)


def _pool(case, seed, g, pages, seqs):
    """A pool whose pages all hold quantised rows, and the 16-bit rings."""
    H, D, top, dtype = case["kv_heads"], case["dim"], TOP[case["code"]], TYPES[case["type"]]
    state = {}
    for n in ("k", "v"):
        x = _rows((pages, H, PAGE // BLOCK, BLOCK, D), dtype, g)
        code, scale = _quantise(x.float(), top)
        state[n] = code.reshape(pages, H, PAGE, D)
        state[n + "_scale"] = scale
        state[n + "_open"] = _rows((seqs, H, RING, D), dtype, g)
    return state


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 17)
    dtype = TYPES[case["type"]]
    if case["op"] == "rope":
        freq, factor = _frequencies(case)
        first = torch.randint(0, case["far"], (1,), device="cuda", generator=g)
        return {"case": case, "q": torch.randn(case["rows"], case["heads"], case["dim"], device="cuda", generator=g).to(dtype),
                "k": torch.randn(case["rows"], case["kv_heads"], case["dim"], device="cuda", generator=g).to(dtype),
                "positions": ((first + torch.arange(case["rows"], device="cuda")) % case["far"]).to(torch.int32),
                "freq": freq.cuda(), "factor": factor}
    lens, new = _lengths(case)
    B, cols = len(lens), max(1, -(-max(lens) // PAGE))
    dst = -(-case["budget"] // PAGE) if case["op"] == "evict" else 0
    pages = B * (cols + dst)
    state = _pool(case, seed, g, pages, B)
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    state.update(case=case, table=order[: B * cols].reshape(B, cols).contiguous(), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                 cu=torch.tensor(cu, dtype=torch.int32, device="cuda"), most=max(new), total=cu[-1])
    if case["op"] == "append":
        state["new_k"] = _rows((cu[-1], case["kv_heads"], case["dim"]), dtype, g)
        state["new_v"] = _rows((cu[-1], case["kv_heads"], case["dim"]), dtype, g)
        # what is read back: from the beginning of the first block that the new rows touch
        begin = [(n - m) // BLOCK * BLOCK for n, m in zip(lens, new)]
        back = [0]
        for n, b in zip(lens, begin):
            back.append(back[-1] + n - b)
        state.update(begin=torch.tensor(begin, dtype=torch.int32, device="cuda"), back=torch.tensor(back, dtype=torch.int32, device="cuda"), back_total=back[-1],
                     back_most=max(n - b for n, b in zip(lens, begin)))
    if case["op"] == "attend":
        state["q"] = torch.randn(cu[-1], case["heads"], case["dim"], device="cuda", generator=g).to(dtype)
        state["scale"] = case["dim"] ** -0.5
        if case["weigh"]:
            state["weight"] = torch.rand(B, case["kv_heads"], cols * PAGE, device="cuda", generator=g) * 4
            state["weight_out"] = torch.zeros(B, case["kv_heads"], cols * PAGE, device="cuda")
    if case["op"] == "evict":
        state["dst_table"] = order[B * cols:].reshape(B, dst).contiguous()
        state["weight"] = torch.rand(B, case["kv_heads"], cols * PAGE, device="cuda", generator=g).pow(4)
        state["begin"] = torch.zeros(B, dtype=torch.int32, device="cuda")
    return state


# ---------------------------------------------------------------- plain forms

def _quantise(x, top):
    """Codes and scales of blocks x [..., 16, D] in 32 bits; a block that holds a value that is not finite reads back as NaN."""
    most = x.abs().amax((-1, -2))
    fine = torch.isfinite(most)
    scale = torch.where(fine, most / top, torch.nan)
    r = x / scale[..., None, None]
    r = torch.where((fine & (most > 0))[..., None, None], r.clamp(-top, top), 0.0)
    return (r.round().to(torch.int8) if top == 127.0 else r.to(torch.float8_e4m3fn)), scale


def _dense(s, name, table, n):
    """The first n rows (a multiple of 64) of each sequence as 32-bit values [B, H, n, D]."""
    at = table[:, : n // PAGE].long()
    code, scale = s[name][at].float(), s[name + "_scale"][at]
    B, P, H, _, D = code.shape
    x = code.reshape(B, P, H, PAGE // BLOCK, BLOCK, D) * scale[..., None, None]
    return x.permute(0, 2, 1, 3, 4, 5).reshape(B, H, n, D)


def _read(s, table, begin, cu, total, most, dtype):
    """Rows begin .. of each sequence, packed: [total, H, D] of keys and of values."""
    row = torch.arange(total, device="cuda")
    seq = torch.searchsorted(cu.long(), row, right=True) - 1
    pos = row - cu[seq].long() + begin[seq].long()
    page = table[seq, pos // PAGE].long()
    out = []
    for name in ("k", "v"):
        code = s[name][page, :, pos % PAGE].float()
        out.append((code * s[name + "_scale"][page, :, pos % PAGE // BLOCK][..., None]).to(dtype))
    return out


def _rope(s):
    c, freq = s["case"], s["freq"]
    half = c["rot"] // 2
    angle = s["positions"].double()[:, None] * freq
    cos, sin = (angle.cos() * s["factor"]).float()[:, None], (angle.sin() * s["factor"]).float()[:, None]

    def turn(x):
        y = x.float()
        rot, rest = y[..., : c["rot"]], y[..., c["rot"]:]
        if c["layout"] == "half":
            a, b = rot[..., :half], rot[..., half:]
            rot = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = rot[..., 0::2], rot[..., 1::2]
            rot = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        return torch.cat([rot, rest], -1).to(x.dtype)

    return {"q": turn(s["q"]), "k": turn(s["k"])}


def _append(s):
    c = s["case"]
    lens, cu, table = s["lens"].long(), s["cu"].long(), s["table"].long()
    new = cu[1:] - cu[:-1]
    start = lens - new
    blocks = (s["most"] + BLOCK - 1) // BLOCK + 1
    at = (start // BLOCK)[:, None] + torch.arange(blocks, device="cuda")  # [B, blocks]
    pos = at[..., None] * BLOCK + torch.arange(BLOCK, device="cuda")  # [B, blocks, 16]
    seq = torch.arange(len(lens), device="cuda")[:, None, None].expand_as(pos)
    is_new, is_old = (pos >= start[:, None, None]) & (pos < lens[:, None, None]), pos < start[:, None, None]
    row = (cu[:-1, None, None] + pos - start[:, None, None]).clamp(0, max(0, s["total"] - 1))
    touched = (at * BLOCK < lens[:, None]) & (new > 0)[:, None]
    b, n = touched.nonzero(as_tuple=True)
    page, slot = table[b, at[b, n] // (PAGE // BLOCK)], at[b, n] % (PAGE // BLOCK)
    keep = is_new & (pos >= (((lens - 1).clamp(min=0) // BLOCK - 1) * BLOCK)[:, None, None])
    for name in ("k", "v"):
        x = torch.where(is_new[..., None, None], s["new_" + name][row], 0)
        x = torch.where(is_old[..., None, None], s[name + "_open"][seq, :, pos % RING], x)  # [B, blocks, 16, H, D]
        code, scale = _quantise(x.float().transpose(2, 3), TOP[c["code"]])  # [B, blocks, H, 16, D]
        s[name + "_scale"][page, :, slot] = scale[b, n]
        H, D = c["kv_heads"], c["dim"]
        bits = s[name].view(torch.uint8).view(-1, H, PAGE // BLOCK, BLOCK, D)
        bits[page, :, slot] = code[b, n].view(torch.uint8)
        bq, nq, iq = keep.nonzero(as_tuple=True)
        s[name + "_open"][bq, :, pos[bq, nq, iq] % RING] = x[bq, nq, iq]
    k, v = _read(s, s["table"], s["begin"], s["back"], s["back_total"], s["back_most"], TYPES[c["type"]])
    return {"k": k, "v": v, "k_open": s["k_open"], "v_open": s["v_open"]}


def _attend(s):
    c = s["case"]
    H, D, Q = c["kv_heads"], c["dim"], s["most"]
    G, B, L = c["heads"] // H, len(s["lens"]), s["table"].shape[1] * PAGE
    cu, lens = s["cu"].long(), s["lens"].long()
    i = torch.arange(Q, device="cuda")
    there = i < (cu[1:] - cu[:-1])[:, None]  # [B, Q]
    row = (cu[:-1, None] + i).clamp(max=max(0, s["total"] - 1))
    q = s["q"][row].float().reshape(B, Q, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * Q, D)
    p = q @ _dense(s, "k", s["table"], L).transpose(-1, -2)
    p = p.reshape(B, H, G, Q, L) * s["scale"]
    at = lens[:, None] - (cu[1:] - cu[:-1])[:, None] + i  # each query's position
    j = torch.arange(L, device="cuda")
    seen = (j <= at[..., None]) & there[..., None]
    if c["window"]:
        seen &= j > at[..., None] - c["window"]
    p = p.masked_fill_(~seen[:, None, None], -torch.inf)
    m = p.amax(-1, keepdim=True)
    m = torch.where(m == -torch.inf, 0.0, m)
    p = p.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    w = torch.where(l > 0, l, 1.0)
    o = (p.reshape(B, H, G * Q, L) @ _dense(s, "v", s["table"], L)).reshape(B, H, G, Q, D) / w
    o = o.permute(0, 3, 1, 2, 4).reshape(B, Q, H * G, D)
    out = {"out": o[there].to(s["q"].dtype)}
    if c["lse"]:
        out["lse"] = (m + l.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(B, Q, H * G)[there]
    if c["weigh"]:
        total = s["weight"] + (p / w).sum((2, 3))
        s["weight_out"].copy_(torch.where(j < lens[:, None, None], total, s["weight_out"]))
        out["weight"] = s["weight_out"]
    return out


def _kept(s):
    """Which positions stay [B, H, budget], in order, -1 past the end."""
    c, lens, w = s["case"], s["lens"].long(), s["weight"]
    L, budget = w.shape[-1], c["budget"]
    j = torch.arange(L, device="cuda")
    n = lens[:, None, None]
    always = (j < c["sinks"]) | (j >= n - c["recent"]) | (n <= budget)
    key = torch.where(always, torch.inf, w)
    key = torch.where(j < n, key, -torch.inf)
    first = key.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    first = torch.where(first < n, first, L).sort(-1).values
    if first.shape[-1] < budget:
        first = torch.nn.functional.pad(first, (0, budget - first.shape[-1]), value=L)
    return torch.where(first < n, first, -1)


def _evict(s):
    c, table, dst = s["case"], s["table"].long(), s["dst_table"].long()
    B, H, D, top = len(s["lens"]), c["kv_heads"], c["dim"], TOP[c["code"]]
    keep = _kept(s)
    budget, cols = keep.shape[-1], dst.shape[1]
    at = torch.nn.functional.pad(keep, (0, cols * PAGE - budget), value=-1).clamp(min=0)
    there = torch.nn.functional.pad(keep, (0, cols * PAGE - budget), value=-1) >= 0  # [B, H, N]
    seq, head = torch.arange(B, device="cuda")[:, None, None], torch.arange(H, device="cuda")[None, :, None]
    page = table[seq, at // PAGE]
    shape = (B, H, cols * (PAGE // BLOCK), BLOCK)
    for name in ("k", "v"):
        code = torch.where(there[..., None], s[name][page, head, at % PAGE].float(), 0.0)
        scale = torch.where(there, s[name + "_scale"][page, head, at % PAGE // BLOCK], 0.0)
        most = (scale * (code.abs().amax(-1) / top)).reshape(shape).amax(-1)  # the new blocks' scales
        ratio = torch.where(most[..., None] > 0, scale.reshape(shape) / most[..., None], 0.0)
        r = (code.reshape(*shape, D) * ratio[..., None]).clamp(-top, top)
        code = r.round().to(torch.int8) if top == 127.0 else r.to(torch.float8_e4m3fn)
        s[name].view(torch.uint8)[dst] = code.view(torch.uint8).reshape(B, H, cols, PAGE, D).transpose(1, 2)
        s[name + "_scale"][dst] = most.reshape(B, H, cols, PAGE // BLOCK).transpose(1, 2)
    weight = torch.where(keep >= 0, s["weight"].gather(-1, keep.clamp(min=0)), 0.0)
    k, v = _read(s, s["dst_table"], s["begin"], s["cu"], s["total"], s["most"], TYPES[c["type"]])
    return {"lens": s["lens"].clamp(max=c["budget"]), "keep": keep.int(), "weight": weight, "k": k, "v": v}


# ---------------------------------------------------------------- the framework's operators

def _package():
    if "qtts_b200" not in sys.modules:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3-tts.cpp_b200")
        at = at if os.path.isdir(at) else os.path.join(os.getcwd(), "qwen3-tts.cpp_b200")
        spec = importlib.util.spec_from_file_location("qtts_b200", os.path.join(at, "__init__.py"), submodule_search_locations=[at])
        module = importlib.util.module_from_spec(spec)
        sys.modules["qtts_b200"] = module
        spec.loader.exec_module(module)
    return sys.modules["qtts_b200"]


def _own(s):
    c, qtts = s["case"], _package()
    if c["op"] == "rope":
        q, k = qtts.rope(s["q"], s["k"], s["positions"], s["freq"], layout=c["layout"], factor=s["factor"])
        return {"q": q, "k": k}
    if "cache" not in s:  # the handle on the pool that a program keeps
        s["cache"] = qtts.KvCache8(s["k"], s["v"], s["k_scale"], s["v_scale"], s["k_open"], s["v_open"])
    cache = s["cache"]
    if c["op"] == "append":
        cache.append(s["new_k"], s["new_v"], s["table"], s["lens"], cu=s["cu"], max_new=s["most"])
        k, v = cache.read(s["table"], s["begin"], s["back"], s["back_total"], max_rows=s["back_most"])
        return {"k": k, "v": v, "k_open": s["k_open"], "v_open": s["v_open"]}
    if c["op"] == "attend":
        out, lse = cache.attend(s["q"], s["table"], s["lens"], cu=s["cu"], max_q=s["most"], scale=s["scale"], window=c["window"],
                                weight=s.get("weight"), weight_out=s.get("weight_out"), want_lse=c["lse"])
        got = {"out": out}
        if c["lse"]:
            got["lse"] = lse
        if c["weigh"]:
            got["weight"] = s["weight_out"]
        return got
    lens, keep, weight = cache.evict(s["table"], s["lens"], s["dst_table"], s["weight"], c["budget"], sinks=c["sinks"], recent=c["recent"])
    k, v = cache.read(s["dst_table"], s["begin"], s["cu"], s["total"], max_rows=s["most"])
    return {"lens": lens, "keep": keep, "weight": weight, "k": k, "v": v}


def run(state):
    if own:
        return _own(state)
    return {"rope": _rope, "append": _append, "attend": _attend, "evict": _evict}[state["case"]["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    D = case["dim"]
    if case["op"] == "rope":
        heads = case["heads"] + case["kv_heads"]
        return {"bytes": case["rows"] * (heads * D * 4 + 4), "flops": case["rows"] * heads * case["rot"] * 3}
    lens, new = _lengths(case)
    H, row = case["kv_heads"], 2 * (D + 4 / BLOCK)  # the bytes of a token's key and value codes and its share of the scales, for one head
    if case["op"] == "append":  # rows in, codes out, codes read back, rows out
        back = sum(n - (n - m) // BLOCK * BLOCK for n, m in zip(lens, new))
        return {"bytes": H * (sum(new) * (4 * D + row) + back * (row + 4 * D)), "flops": 4 * H * D * sum(new)}
    if case["op"] == "attend":
        pairs = read = 0
        for n, m in zip(lens, new):
            window = case["window"] or n + m
            for at in range(n - m, n):
                pairs += max(0, min(at + 1, window))
            read += min(n, window + m - 1)
        weigh = 8 * H * sum(lens) if case["weigh"] else 0
        return {"bytes": H * read * row + sum(new) * case["heads"] * (D * 4 + (4 if case["lse"] else 0)) + weigh, "flops": 4 * D * case["heads"] * pairs}
    # the weights, the kept rows' codes in and out, the codes read back, the rows out
    return {"bytes": H * (4 * sum(lens) + sum(new) * (3 * row + 4 * D + 12)), "flops": 4 * H * D * sum(new)}


# ---------------------------------------------------------------- the definition, in 64 bits

def _exact_blocks(x, top):
    """Values of blocks [..., 16, D] in 64 bits after their quantisation."""
    scale = x.abs().amax((-1, -2), keepdim=True) / top
    code = torch.where(scale > 0, x / scale, torch.zeros_like(x))
    return _exact_code(code, top) * scale


def _exact_code(r, top):
    r = r.clamp(-top, top)
    if top == 127.0:
        return torch.round(r)
    # 8-bit floats: 3 bits of mantissa, exponents down to -6
    e = torch.floor(torch.log2(r.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(r / step) * step


def _exact_value(s, name, table, b, n):
    """The first n rows of sequence b, [H, n, D], in 64 bits."""
    rows = torch.cat([s[name][int(p)].double() for p in table[b, : -(-n // PAGE)].tolist()], 1)[:, :n]
    scale = torch.cat([s[name + "_scale"][int(p)].double() for p in table[b, : -(-n // PAGE)].tolist()], 1)
    return rows * scale.repeat_interleave(BLOCK, 1)[:, :n, None]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        turns = s["positions"].double()[:, None] * s["freq"]
        unit = torch.polar(torch.full_like(turns, s["factor"]), turns)[:, None]
        got = {}
        for name in ("q", "k"):
            x = s[name].double()
            pair = x[..., : case["rot"]].unflatten(-1, (2, -1)).transpose(-1, -2) if case["layout"] == "half" else x[..., : case["rot"]].unflatten(-1, (-1, 2))
            z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * unit)
            z = z.transpose(-1, -2) if case["layout"] == "half" else z
            got[name] = torch.cat([z.flatten(-2), x[..., case["rot"]:]], -1)
        return got
    lens, new = _lengths(case)
    top, B, H, D = TOP[case["code"]], len(lens), case["kv_heads"], case["dim"]
    if sum(lens) * H > 3000000 or (case["op"] == "attend" and work(case)["flops"] > 3e12):
        return None
    cu = s["cu"].tolist()
    if case["op"] == "append":
        got = {"k": [], "v": []}
        for name in ("k", "v"):
            ring = s[name + "_open"].double()
            for b in range(B):
                n, m = lens[b], new[b]
                begin = (n - m) // BLOCK * BLOCK
                if m == 0:
                    # untouched: what the pages held
                    got[name].append(_exact_value(s, name, s["table"], b, n)[:, begin:].transpose(0, 1))
                    continue
                old = ring[b][:, torch.arange(begin, n - m, device="cuda") % RING]
                x = torch.cat([old, s["new_" + name][cu[b]: cu[b + 1]].double().transpose(0, 1)], 1)
                pad = torch.nn.functional.pad(x, (0, 0, 0, -x.shape[1] % BLOCK))
                y = _exact_blocks(pad.reshape(H, -1, BLOCK, D), top).reshape(H, -1, D)[:, : n - begin]
                got[name].append(y.transpose(0, 1))
                for p in range(max(n - m, ((n - 1) // BLOCK - 1) * BLOCK), n):
                    ring[b][:, p % RING] = x[:, p - begin]
            got[name + "_open"] = ring
        return {"k": torch.cat(got["k"]), "v": torch.cat(got["v"]), "k_open": got["k_open"], "v_open": got["v_open"]}
    if case["op"] == "attend":
        outs, lses = [], []
        weight = None if not case["weigh"] else s["weight_out"].double()
        G = case["heads"] // H
        for b in range(B):
            n, m = lens[b], new[b]
            out = torch.zeros(m, H, G, D, dtype=torch.float64, device="cuda")
            lse = torch.full((m, H, G), -torch.inf, dtype=torch.float64, device="cuda")
            if weight is not None:
                weight[b, :, :n] = s["weight"][b, :, :n].double()
            if n and m:
                k, v = _exact_value(s, "k", s["table"], b, n), _exact_value(s, "v", s["table"], b, n)
                q = s["q"][cu[b]: cu[b + 1]].double().reshape(m, H, G, D)
                at = torch.arange(n - m, n, device="cuda")[:, None]
                j = torch.arange(n, device="cuda")
                hidden = (j > at) | (j <= at - (case["window"] or n + m))
                for h in range(H):
                    for g in range(G):
                        z = ((q[:, h, g] @ k[h].T) * s["scale"]).masked_fill(hidden, -torch.inf)
                        lse[:, h, g] = z.logsumexp(-1)
                        p = (z - lse[:, h, g, None]).exp().nan_to_num(0.0)
                        out[:, h, g] = p @ v[h]
                        if weight is not None:
                            weight[b, h, :n] += p.sum(0)
            outs.append(out.reshape(m, H * G, D))
            lses.append(lse.reshape(m, H * G))
        got = {"out": torch.cat(outs)}
        if case["lse"]:
            got["lse"] = torch.cat(lses)
        if weight is not None:
            got["weight"] = weight
        return got
    budget = case["budget"]
    keep = torch.full((B, H, budget), -1, dtype=torch.int32, device="cuda")
    weight = torch.zeros(B, H, budget, dtype=torch.float64, device="cuda")
    rows = {"k": [], "v": []}
    heavy = s["weight"].cpu().numpy()
    for b in range(B):
        n, m = lens[b], new[b]
        for h in range(H):
            if n <= budget:
                at = list(range(n))
            else:
                middle = range(case["sinks"], n - case["recent"])
                chosen = sorted(middle, key=lambda i: (-heavy[b, h, i], i))[: budget - case["sinks"] - case["recent"]]
                at = sorted(chosen) + list(range(case["sinks"])) + list(range(n - case["recent"], n))
                at.sort()
            keep[b, h, :m] = torch.tensor(at, dtype=torch.int32, device="cuda")
        weight[b, :, :m] = s["weight"][b].gather(-1, keep[b, :, :m].long()).double()
        for name in ("k", "v"):
            if not m:
                rows[name].append(torch.zeros(0, H, D, dtype=torch.float64, device="cuda"))
                continue
            x = _exact_value(s, name, s["table"], b, n).gather(1, keep[b, :, :m].long()[..., None].expand(-1, -1, D))
            x = torch.nn.functional.pad(x, (0, 0, 0, -m % BLOCK))
            rows[name].append(_exact_blocks(x.reshape(H, -1, BLOCK, D), top).reshape(H, -1, D)[:, :m].transpose(0, 1))
    return {"lens": s["lens"].clamp(max=budget), "keep": keep, "weight": weight, "k": torch.cat(rows["k"]), "v": torch.cat(rows["v"])}
