"""A prompt's tokens over the page pool of a batch, operator by operator, as cases to be timed and compared.

A server that holds many sequences in one pool of pages runs prompts whole or in chunks, drafts that are to be verified, and
steps in which some sequences bring a chunk and others one token. Per step it takes pages for the new tokens and
gives back those of sequences that ended or were cut (`reserve`: page tables, first rows, and each row's sequence and
slot), per layer it puts the rows' keys and values into the pool (`append`: norm, rotation, cache rows) and attends from
every row to its own sequence's slots up to its own (`attend`).

Sizes are those of this repository's models (heads 32/8, 16/8 and 40/8 of 128) and generic ones. Counts and lengths of a
batch spread evenly between two bounds, in an order drawn from the seed.
"""
import ctypes
import math
import os
import sys

import numpy as np
import torch

own = False
PAGE = 64   # positions per page


# ------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one draft of five tokens verified in a long chat, the smallest call: latency counts
        {"name": "attend-5-at-7000", "kind": "attend", "B": 1, "c_lo": 5, "c_hi": 5, "mixed": False, "lo": 7000, "hi": 7000, "heads": 32,
         "kv_heads": 8, "dim": 128, "half": "bf16", "io": "fp32", "window": 0},
        # a whole prompt, activations in the cache's type
        {"name": "attend-2048-at-0", "kind": "attend", "B": 1, "c_lo": 2048, "c_hi": 2048, "mixed": False, "lo": 0, "hi": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "half": "bf16", "io": "half", "window": 0},
        # a chunk far into a long document
        {"name": "attend-2048-at-30000", "kind": "attend", "B": 1, "c_lo": 2048, "c_hi": 2048, "mixed": False, "lo": 30000, "hi": 30000, "heads": 40,
         "kv_heads": 8, "dim": 128, "half": "bf16", "io": "half", "window": 0},
        # a server's mixed step: every fourth sequence brings a chunk, the others one token
        {"name": "attend-32-mixed-7k", "kind": "attend", "B": 32, "c_lo": 33, "c_hi": 400, "mixed": True, "lo": 0, "hi": 7000, "heads": 32,
         "kv_heads": 8, "dim": 128, "half": "bf16", "io": "half", "window": 0},
        # chunks of several prompts with this framework's own fp32 activations
        {"name": "attend-6-ragged-fp32", "kind": "attend", "B": 6, "c_lo": 77, "c_hi": 611, "mixed": False, "lo": 0, "hi": 3001, "heads": 40,
         "kv_heads": 8, "dim": 128, "half": "bf16", "io": "fp32", "window": 0},
        # sliding-window layers with half-size heads over an f16 cache, some sequences idle
        {"name": "attend-24-window-f16", "kind": "attend", "B": 24, "c_lo": 0, "c_hi": 300, "mixed": False, "lo": 5, "hi": 16000, "heads": 16,
         "kv_heads": 8, "dim": 64, "half": "f16", "io": "half", "window": 1024},
        # the draft's keys and values: nothing but latency
        {"name": "append-5", "kind": "append", "B": 1, "c_lo": 5, "c_hi": 5, "lo": 7000, "hi": 7000, "heads": 32, "kv_heads": 8, "dim": 128,
         "half": "bf16", "io": "fp32", "rot": 128, "pairs": "halves", "scaled": False, "norm": True, "positions": False},
        # a whole prompt's
        {"name": "append-2048", "kind": "append", "B": 1, "c_lo": 2048, "c_hi": 2048, "lo": 0, "hi": 0, "heads": 32, "kv_heads": 8, "dim": 128,
         "half": "bf16", "io": "half", "rot": 128, "pairs": "halves", "scaled": False, "norm": True, "positions": False},
        # chunks of several sequences whose slots are no positions, neighbours rotated, half of the head, frequencies scaled for far positions
        {"name": "append-24-scaled-f16", "kind": "append", "B": 24, "c_lo": 1, "c_hi": 333, "lo": 0, "hi": 2000, "heads": 40, "kv_heads": 8, "dim": 128,
         "half": "f16", "io": "fp32", "rot": 64, "pairs": "neighbours", "scaled": True, "norm": False, "positions": True},
        # a decode step: one more token for each, a page now and then
        {"name": "reserve-32-step", "kind": "reserve", "B": 32, "hi": 8191, "grow": 1, "ended": 0.0, "short": False},
        # prompts arrive where others end
        {"name": "reserve-200-prompts", "kind": "reserve", "B": 200, "hi": 4096, "grow": 300, "ended": 0.2, "short": False},
        # a very large batch whose pool runs out
        {"name": "reserve-4000-short", "kind": "reserve", "B": 4000, "hi": 3000, "grow": 40, "ended": 0.1, "short": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "reserve"])
    if kind == "reserve":
        return {"kind": kind, "B": _log(rng, 1, 4000), "hi": _log(rng, 1, 8191), "grow": _log(rng, 1, 300), "ended": rng.choice([0.0, 0.1, 0.3]),
                "short": rng.random() < 0.3}
    kv, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128])
    heads = kv * rng.choice([1, 2, 4, 5, 8, 16] if kv <= 2 else [1, 2, 4, 5])
    c = {"kind": kind, "heads": heads, "kv_heads": kv, "dim": dim, "half": rng.choice(["bf16", "bf16", "f16"]), "io": rng.choice(["fp32", "half"])}
    B = _log(rng, 1, 48)
    most = min(_log(rng, 1, 2048), 8000 // B)
    if kind == "append":
        return {**c, "B": B, "c_lo": rng.randint(0, most), "c_hi": most, "lo": 0, "hi": _log(rng, 1, 4000), "rot": rng.choice([dim, dim, dim // 2]),
                "pairs": rng.choice(["halves", "neighbours"]), "scaled": rng.random() < 0.5, "norm": rng.random() < 0.5, "positions": rng.random() < 0.5}
    # no more scores than the largest listed case has, no more slots than a few long documents
    hi = max(0, min(_log(rng, 1, 131072), min(300000 // B, 2_600_000_000 // (B * heads * most)) - most))
    return {**c, "B": B, "c_lo": rng.randint(0, most), "c_hi": most, "mixed": rng.random() < 0.4, "lo": rng.randint(0, hi), "hi": hi,
            "window": rng.choice([0, 0, _log(rng, 1, 4096)])}


def _spread(c, lo, hi, order):
    n = c["B"]
    return [hi - (hi - lo) * (order(i) % n) // max(1, n - 1) for i in range(n)]


def _batch(c):
    """New tokens and earlier slots of each sequence, in an order that the seed permutes."""
    counts, before = _spread(c, c["c_lo"], c["c_hi"], lambda i: i), _spread(c, c["lo"], c["hi"], lambda i: 5 * i + 3)
    if c.get("mixed"):
        counts = [x if i % 4 == 0 else 1 for i, x in enumerate(counts)]
    return np.array(counts, np.int64), np.array(before, np.int64)


def _asked(c):
    """Lengths and wanted lengths of a reservation."""
    n, lens = c["B"], np.array(_spread(c, 0, c["hi"], lambda i: 5 * i + 3), np.int64)
    add = np.array(_spread(c, min(1, c["grow"]), c["grow"], lambda i: 3 * i), np.int64)
    ended = (np.arange(n) * 0.618034) % 1.0 < c["ended"]
    return lens, np.where(ended, np.where(np.arange(n) % 3 == 0, lens // 2, 0), lens + add)


def _pages(x):
    return -(-x // PAGE)


def _pool_pages(c):
    lens, want = _asked(c)
    used, more = int(_pages(lens).sum()), int(np.maximum(0, _pages(want) - _pages(lens)).sum())
    back = int(np.maximum(0, _pages(lens) - _pages(want)).sum())
    return used, max(1, more * 2 // 3 - back) if c["short"] else more + 7


def work(c):
    if c["kind"] == "reserve":
        lens, want = _asked(c)
        moved = int(np.abs(_pages(want) - _pages(lens)).sum())
        return {"bytes": 20.0 * c["B"] + 8.0 * moved + 8.0 * int(np.maximum(0, want - lens).sum()), "flops": 0.0}
    counts, before = _batch(c)
    n, d, H, rows, out = c["kv_heads"], c["dim"], c["heads"], int(counts.sum()), 4.0 if c["io"] == "fp32" else 2.0
    if c["kind"] == "append":
        return {"bytes": rows * d * (4.0 * (H + 2 * n) + out * H + 4.0 * n), "flops": 6.0 * rows * d * (H + n)}
    far, pairs, seen = c["window"] or 1 << 60, 0, 0
    for x, p in zip(counts, before):
        pairs += int(np.minimum(p + 1 + np.arange(x), far).sum())
        seen += int(min(p + x, far + x - 1)) if x else 0
    return {"bytes": 4.0 * n * d * seen + 2.0 * out * rows * H * d, "flops": 4.0 * H * d * pairs}


# ------------------------------------------------------------------------------------------- inputs
def _half(c):
    return torch.bfloat16 if c["half"] == "bf16" else torch.float16


def _ints(x):
    return torch.tensor(np.ascontiguousarray(x), dtype=torch.int32, device="cuda")


def _tables(lens, width, order):
    """A page table over distinct pages in the given order; entries behind a sequence's last page name none."""
    used = _pages(lens)
    table = np.full((len(lens), width), -1, np.int64)
    at = np.concatenate([[0], np.cumsum(used)])
    for b in range(len(lens)):
        table[b, :used[b]] = order[at[b]:at[b + 1]]
    return table


def _frequencies(c):
    """Inverse frequencies of the rotated pairs and the factor of their sines: as they are, or low ones stretched 16 times with a ramp between."""
    rot, base = c["rot"], 1e6
    f = base ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)
    if not c["scaled"]:
        return f, 1.0
    factor, trained = 16.0, 8192.0
    turns = trained * f / (2 * math.pi)                        # of each pair within the trained length
    keep = np.clip((turns - 1.0) / (32.0 - 1.0), 0.0, 1.0)
    return f * keep + f / factor * (1.0 - keep), 0.1 * math.log(factor) + 1.0


def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rs = np.random.default_rng(seed)
    randn = lambda *shape: torch.randn(shape, device="cuda", generator=gen)  # noqa: E731
    s = dict(c)
    if c["kind"] == "reserve":
        lens, want = _asked(c)
        by = rs.permutation(c["B"])
        lens, want = lens[by], want[by]
        used, free = _pool_pages(c)
        order = rs.permutation(used + free)
        s["max_len"] = int(max(1, lens.max(), want.max()))
        s["n_pages"], s["rows"] = used + free, int(np.maximum(0, want - lens).sum())
        stack = np.full(used + free, -1, np.int64)
        stack[:free] = order[used:]
        s["table"], s["len"], s["want"] = _ints(_tables(lens, _pages(s["max_len"]), order)), _ints(lens), _ints(want)
        s["free"], s["n_free"] = _ints(stack), _ints([free])
        s["len_out"], s["n_free_out"], s["start"], s["count"] = (torch.zeros(x, dtype=torch.int32, device="cuda") for x in (c["B"], 1, c["B"], c["B"]))
        s["seq"], s["slot"] = (torch.zeros(max(1, s["rows"]), dtype=torch.int32, device="cuda") for _ in range(2))
        return s
    counts, before = _batch(c)
    by = rs.permutation(c["B"])
    counts, before = counts[by], before[by]
    lens = counts + before
    n, d, H, rows = c["kv_heads"], c["dim"], c["heads"], max(1, int(counts.sum()))
    s["max_len"], s["rows"] = max(1, int(lens.max())), rows
    pages = max(1, int(_pages(lens).sum()))
    s["k"], s["v"] = (torch.randn((pages, n, PAGE, d), device="cuda", generator=gen, dtype=_half(c)) for _ in range(2))
    s["table"] = _ints(_tables(lens, _pages(s["max_len"]), rs.permutation(pages)))
    s["len"], s["count"], s["start"] = _ints(lens), _ints(counts), _ints(np.cumsum(counts) - counts)
    io = torch.float32 if c["io"] == "fp32" else _half(c)
    if c["kind"] == "attend":
        s["q"], s["scale"] = (2.0 * randn(rows, H * d)).to(io), d ** -0.5
        s["most"] = int(counts.max())
        s["out"] = torch.zeros(rows, H * d, device="cuda", dtype=io)
        return s
    seq = np.repeat(np.arange(c["B"]), counts)
    slot = np.concatenate([np.arange(p, p + x) for p, x in zip(before, counts)]) if counts.sum() else np.zeros(0, np.int64)
    if not counts.sum():
        seq, slot = np.array([-1]), np.array([-1])             # a row that holds no token
    s["seq"], s["slot"] = _ints(seq), _ints(slot)
    s["pos"] = _ints(slot + rs.integers(0, 100000, c["B"])[np.maximum(seq, 0)]) if c["positions"] else None
    f, s["rope_scale"] = _frequencies(c)
    s["inv_freq"] = torch.tensor(f, dtype=torch.float32, device="cuda")
    s["qkv"] = randn(rows, (H + 2 * n) * d)
    s["qn"], s["kn"] = (1.0 + 0.1 * randn(d), 1.0 + 0.1 * randn(d)) if c["norm"] else (None, None)
    s["q"] = torch.zeros(rows, H * d, device="cuda", dtype=io)
    return s


# ------------------------------------------------------------------------------------------- plain forms
def _gather(pool, table, count):
    """Slots 0 .. count - 1 of every sequence, as [B][heads][count][dim] in 32 bits."""
    x = pool[table.long().clamp(min=0)].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])[:, :, :count].float()


def _plain_attend(s):
    B, H, n, d, top, C = s["B"], s["heads"], s["kv_heads"], s["dim"], s["max_len"], s["most"]
    count, start, ln = s["count"].long(), s["start"].long(), s["len"].long()
    row = (start[:, None] + torch.arange(C, device="cuda")).clamp(max=s["rows"] - 1)
    at = (ln - count)[:, None] + torch.arange(C, device="cuda")               # [B][C]: each query's own slot
    slot = torch.arange(top, device="cuda")
    seen = (slot <= at[..., None]) & (slot < ln[:, None, None])
    if s["window"]:
        seen &= slot > at[..., None] - s["window"]
    q = (s["q"][row].float() * s["scale"]).view(B, C, n, H // n, d).permute(0, 2, 3, 1, 4).reshape(B, n, H // n * C, d).contiguous()
    k, v = _gather(s["k"], s["table"], top), _gather(s["v"], s["table"], top)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).view(B, n, H // n, C, top)
    score.masked_fill_(~seen[:, None, None], -math.inf)
    most = score.amax(-1, keepdim=True)
    e = score.sub_(torch.where(most == -math.inf, torch.zeros_like(most), most)).exp_()
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(B, n, H // n * C, top), v).view(B, n, H // n, C, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 3, 1, 2, 4).reshape(B, C, H * d)
    r = torch.arange(s["rows"], device="cuda")
    b = torch.searchsorted(start + count, r, right=True).clamp(max=B - 1)
    mine = o[b, (r - start[b]).clamp(0, C - 1)].to(s["out"].dtype)
    s["out"].copy_(torch.where((r < start[b] + count[b])[:, None], mine, s["out"]))
    return {"out": s["out"]}


def _plain_append(s):
    R, H, n, d, rot = s["rows"], s["heads"], s["kv_heads"], s["dim"], s["rot"]
    on = s["seq"] >= 0
    x = s["qkv"].view(R, H + 2 * n, d)
    qk = x[:, :H + n]
    if s["qn"] is not None:
        w = torch.cat([s["qn"].expand(H, d), s["kn"].expand(n, d)])
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + 1e-6) * w
    pos = s["slot"] if s["pos"] is None else s["pos"]
    angle = pos.double()[:, None] * s["inv_freq"].double()                    # far positions: 32 bits lose the angle
    cos, sin = ((f(angle) * s["rope_scale"]).float()[:, None] for f in (torch.cos, torch.sin))
    if s["pairs"] == "halves":
        a, b = qk[..., :rot // 2], qk[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = qk[..., 0:rot:2], qk[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    qk = torch.cat([turned, qk[..., rot:]], -1)
    s["q"].copy_(torch.where(on[:, None], qk[:, :H].reshape(R, H * d).to(s["q"].dtype), s["q"]))
    slot, seq = s["slot"].long().clamp(min=0), s["seq"].long().clamp(min=0)
    page = s["table"].long()[seq, slot // PAGE].clamp(min=0)
    for pool, new in ((s["k"], qk[:, H:]), (s["v"], x[:, H + n:])):
        pool[page, :, slot % PAGE] = torch.where(on[:, None, None], new.to(pool.dtype), pool[page, :, slot % PAGE])
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _plain_reserve(s):
    B, R, N, P = s["B"], s["rows"], s["n_pages"], s["table"].shape[1]
    ln, want = s["len"].long().clamp(0, s["max_len"]), s["want"].long().clamp(0, s["max_len"])
    have, aim = -(-ln // PAGE), -(-want // PAGE)
    entry = torch.arange(P, device="cuda")
    flat = s["table"].reshape(-1).long()
    back = ((entry >= aim[:, None]) & (entry < have[:, None])).reshape(-1) & (flat >= 0) & (flat < N)
    nf = s["n_free"].long().clamp(0, N)
    place = nf + back.long().cumsum(0) - 1                                    # of each page that comes back
    free = torch.cat([s["free"].long(), torch.zeros(1, dtype=torch.long, device="cuda")])
    free = free.scatter(0, torch.where(back & (place < N), place, N), torch.where(back, flat, torch.zeros_like(flat)))
    nf = (nf + back.sum()).clamp(max=N)
    add, need = (want - ln).clamp(min=0), torch.where(want > ln, aim - have, 0)
    upto, start = need.cumsum(0), add.cumsum(0) - add
    granted = (add > 0) & (start + add <= R) & ((need == 0) | (upto <= nf))
    took = torch.where(granted, need, 0)
    first = took.cumsum(0) - took
    new = (entry >= have[:, None]) & (entry < (have + took)[:, None])
    which = nf - 1 - (first[:, None] + entry - have[:, None])
    s["table"].copy_(torch.where(new, free[which.clamp(0, N)].to(torch.int32), s["table"]))
    s["free"].copy_(free[:N])
    s["n_free_out"].copy_(nf - took.sum())
    s["len_out"].copy_(torch.where(granted | (want < ln), want, ln))
    s["count"].copy_(torch.where(granted, add, 0))
    s["start"].copy_(start)
    r = torch.arange(R, device="cuda")
    b = torch.searchsorted(start + add, r, right=True).clamp(max=B - 1)
    on = granted[b] & (r < start[b] + add[b])
    s["seq"][:R].copy_(torch.where(on, b, -1))
    s["slot"][:R].copy_(torch.where(on, ln[b] + r - start[b], -1))
    return _reserved(s)


def _reserved(s):
    return {x: s[x] for x in ("table", "free", "n_free_out", "len_out", "start", "count", "seq", "slot")}


# ------------------------------------------------------------------------------------------- the framework's calls
def _ptr(t):
    return None if t is None else t.data_ptr()


def _calls(s):
    """What a program sets up once for its buffers: the cache's description, the workspace and the bound call."""
    at = os.path.join(os.getcwd(), "mlx-runner_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import mlxr
    lib = mlxr.lib
    stream = torch.cuda.current_stream().cuda_stream

    def work(bytes_):
        s["work"] = torch.zeros(max(16, bytes_), dtype=torch.uint8, device="cuda")
        return s["work"].data_ptr(), s["work"].numel()

    if s["kind"] == "reserve":   # no keys or values are touched: the pool is anything aligned on the device
        pool, n_pages, n, d, st = s["free"], s["n_pages"], 1, 64, 0
    else:
        pool, n_pages, n, d, st = s["k"], s["k"].shape[0], s["kv_heads"], s["dim"], int(s["half"] == "f16")
    kv = mlxr.PagedKV(k=_ptr(pool), v=_ptr(s.get("v", pool)), table=_ptr(s["table"]), len=_ptr(s["len"]), weight=None, position=None, n_pages=n_pages,
                      table_stride=s["table"].shape[1], slot_stride=0, max_len=s["max_len"], B=s["B"], nKV=n, D=d, st=st)
    ref = ctypes.byref(kv)
    s["kv"], io = kv, int(s.get("io") == "half")
    if s["kind"] == "reserve":
        call, args = lib.mlxr_k_paged_reserve, (ref, _ptr(s["want"]), _ptr(s["free"]), _ptr(s["n_free"]), s["rows"], _ptr(s["len_out"]), _ptr(s["n_free_out"]),
                                                _ptr(s["start"]), _ptr(s["count"]), _ptr(s["seq"]), _ptr(s["slot"]),
                                                *work(lib.mlxr_k_paged_reserve_work(ref, s["rows"])), stream)
    elif s["kind"] == "append":
        call, args = lib.mlxr_k_paged_append_rows, (ref, _ptr(s["qkv"]), s["qkv"].shape[1], s["rows"], _ptr(s["seq"]), _ptr(s["slot"]), _ptr(s["pos"]),
                                                    _ptr(s["inv_freq"]), s["rope_scale"], _ptr(s["qn"]), _ptr(s["kn"]), s["heads"], s["rot"],
                                                    int(s["pairs"] == "neighbours"), 1e-6, _ptr(s["q"]), io, s["heads"] * s["dim"], stream)
    else:
        width = s["heads"] * s["dim"]
        call, args = lib.mlxr_k_paged_attention_rows, (ref, _ptr(s["start"]), _ptr(s["count"]), s["rows"], _ptr(s["q"]), io, width, s["heads"], s["window"],
                                                       s["scale"], _ptr(s["out"]), width,
                                                       *work(lib.mlxr_k_paged_attention_rows_work(ref, s["heads"], s["rows"], io)), stream)
    return lambda: mlxr.check(call(*args))


def run(s):
    kind = s["kind"]
    if own:
        if "call" not in s:
            s["call"] = _calls(s)
        s["call"]()
        if kind == "attend":
            return {"out": s["out"]}
        return {"q": s["q"], "k": s["k"], "v": s["v"]} if kind == "append" else _reserved(s)
    return {"attend": _plain_attend, "append": _plain_append, "reserve": _plain_reserve}[kind](s)


# ------------------------------------------------------------------------------------------- the definition in 64 bits
def _exact_attend(s):
    H, n, d = s["heads"], s["kv_heads"], s["dim"]
    G = H // n
    out = s["out"].double().view(-1, H, d)
    for b, (count, length) in enumerate(zip(s["count"].tolist(), s["len"].tolist())):
        if count == 0:
            continue
        first, at = int(s["start"][b]), torch.arange(length - count, length, device="cuda")
        low = max(0, length - count + 1 - s["window"]) if s["window"] else 0
        pages, slot = s["table"][b, :_pages(length)].long(), torch.arange(low, length, device="cuda")
        hidden = slot > at[:, None]
        if s["window"]:
            hidden |= slot <= at[:, None] - s["window"]
        for h in range(n):
            k, v = (s[x][pages, h].reshape(-1, d)[low:length].double() for x in ("k", "v"))
            for g in range(h * G, h * G + G):
                q = s["q"][first:first + count].view(count, H, d)[:, g].double()
                p = torch.softmax((q @ k.t().contiguous() * float(s["scale"])).masked_fill_(hidden, -math.inf), 1)
                out[first:first + count, g] = p @ v
    return {"out": out.view(-1, H * d)}


def _exact_append(s):
    R, H, n, d, rot = s["rows"], s["heads"], s["kv_heads"], s["dim"], s["rot"]
    x = s["qkv"].cpu().double().numpy().reshape(R, H + 2 * n, d)
    heads = x[:, :H + n].copy()
    if s["qn"] is not None:
        heads /= np.sqrt((heads ** 2).mean(-1, keepdims=True) + 1e-6)
        heads[:, :H] *= s["qn"].cpu().double().numpy()
        heads[:, H:] *= s["kn"].cpu().double().numpy()
    pos = (s["slot"] if s["pos"] is None else s["pos"]).cpu().numpy()
    turn = float(s["rope_scale"]) * np.exp(1j * pos[:, None] * s["inv_freq"].cpu().double().numpy())[:, None]
    i, j = (np.arange(rot // 2), np.arange(rot // 2, rot)) if s["pairs"] == "halves" else (np.arange(0, rot, 2), np.arange(1, rot, 2))
    z = (heads[..., i] + 1j * heads[..., j]) * turn
    heads[..., i], heads[..., j] = z.real, z.imag
    q, k, v = s["q"].cpu().double(), s["k"].cpu().double(), s["v"].cpu().double()
    table = s["table"].cpu().numpy()
    for r, (b, t) in enumerate(zip(s["seq"].tolist(), s["slot"].tolist())):
        if b < 0:
            continue
        q[r] = torch.from_numpy(heads[r, :H].reshape(-1))
        k[table[b, t // PAGE], :, t % PAGE] = torch.from_numpy(heads[r, H:])
        v[table[b, t // PAGE], :, t % PAGE] = torch.from_numpy(x[r, H + n:])
    return {"q": q, "k": k, "v": v}


def _exact_reserve(s):
    """Page by page and sequence by sequence, as one would on paper."""
    found = {x: s[x].cpu().numpy().copy() for x in ("table", "free", "len", "want", "seq", "slot")}
    table, free, lens, want = (found[x] for x in ("table", "free", "len", "want"))
    nf, N, R = int(s["n_free"][0]), s["n_pages"], s["rows"]
    for b in range(s["B"]):
        for e in range(_pages(int(want[b])), _pages(int(lens[b]))):
            if 0 <= table[b, e] < N and nf < N:
                free[nf] = table[b, e]
                nf += 1
    start, count, len_out = (np.zeros(s["B"], np.int64) for _ in range(3))
    found["seq"][:R], found["slot"][:R] = -1, -1
    row, top, asked = 0, nf, 0
    for b in range(s["B"]):
        start[b], len_out[b] = row, min(lens[b], want[b])
        more = int(want[b]) - int(lens[b])
        if more <= 0:
            continue
        entries = range(_pages(int(lens[b])), _pages(int(want[b])))
        asked += len(entries)
        if row + more <= R and (len(entries) == 0 or asked <= top):
            for e in entries:
                nf -= 1
                table[b, e] = free[nf]
            len_out[b], count[b] = want[b], more
            found["seq"][row:row + more], found["slot"][row:row + more] = b, np.arange(lens[b], want[b])
        row += more
    return {"table": table, "free": free, "n_free_out": np.array([nf]), "len_out": len_out, "start": start, "count": count, "seq": found["seq"], "slot": found["slot"]}


def exact(c, seed):
    return {"attend": _exact_attend, "append": _exact_append, "reserve": _exact_reserve}[c["kind"]](prepare(c, seed))
