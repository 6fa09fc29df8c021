"""One decode step of a batch of sequences, operator by operator, as cases to be timed and compared.

A server that decodes many sequences at once holds their keys and values in one pool of pages. Per layer and
step it appends the new tokens' keys and values, attends with one query token per sequence (keeping, where the
cache has a budget, how much attention each slot has drawn), and now and then moves the slots that drew most
into fewer pages; after the last layer it draws each sequence's token. These are the four operators here.

Sizes are those of this repository's models (heads 32/8, 16/8 and 40/8 of 128, vocabularies 151936 and 128256)
and generic ones. The lengths of a batch spread evenly between two bounds, in an order drawn from the seed.
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
        # one chat at a usual context, the smallest step: latency counts
        {"name": "attend-1x4096", "kind": "attend", "B": 1, "lo": 4096, "hi": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "half": "bf16",
         "window": 0, "weights": False},
        # a server's batch: chats of every length, an idle row among them
        {"name": "attend-32-ragged-8k", "kind": "attend", "B": 32, "lo": 0, "hi": 8191, "heads": 32, "kv_heads": 8, "dim": 128, "half": "bf16",
         "window": 0, "weights": False},
        # few long documents
        {"name": "attend-4-long-128k", "kind": "attend", "B": 4, "lo": 98765, "hi": 131072, "heads": 40, "kv_heads": 8, "dim": 128,
         "half": "bf16", "window": 0, "weights": False},
        # the same batch under a cache budget: every slot's weight is kept
        {"name": "attend-16-weights-4k", "kind": "attend", "B": 16, "lo": 700, "hi": 4100, "heads": 40, "kv_heads": 8, "dim": 128, "half": "bf16",
         "window": 0, "weights": True},
        # sliding-window layers with half-size heads over an f16 cache
        {"name": "attend-24-window-f16", "kind": "attend", "B": 24, "lo": 5, "hi": 16000, "heads": 16, "kv_heads": 8, "dim": 64, "half": "f16",
         "window": 1024, "weights": False},
        # one sequence's append: nothing but latency
        {"name": "append-1", "kind": "append", "B": 1, "heads": 32, "kv_heads": 8, "dim": 128, "half": "bf16", "rot": 128, "far": 4095, "norm": True},
        # a full server's append at far positions, partly rotated, no q/k norm
        {"name": "append-200-f16", "kind": "append", "B": 200, "heads": 40, "kv_heads": 8, "dim": 128, "half": "f16", "rot": 64, "far": 131071,
         "norm": False},
        # one sequence reaches twice its budget
        {"name": "evict-1-4096-to-2048", "kind": "evict", "B": 1, "lo": 4096, "hi": 4096, "kv_heads": 8, "dim": 128, "half": "bf16",
         "budget": 2048, "sink": 4, "window": 512},
        # a batch of long sequences cut to a quarter, those below the budget moved whole
        {"name": "evict-24-ragged-16k", "kind": "evict", "B": 24, "lo": 100, "hi": 16001, "kv_heads": 8, "dim": 128, "half": "bf16",
         "budget": 4000, "sink": 4, "window": 500},
        # one chat's token with this repository's default parameters
        {"name": "sample-1", "kind": "sample", "rows": 1, "vocab": 151936, "mix": "default"},
        # a server's rows, each with its request's parameters (greedy, top-k, top-p, min-p, none)
        {"name": "sample-256-mixed", "kind": "sample", "rows": 256, "vocab": 151936, "mix": "mixed"},
        # rows that only cut the tail by mass
        {"name": "sample-33-top-p", "kind": "sample", "rows": 33, "vocab": 128256, "mix": "top-p"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "append", "evict", "sample"])
    if kind == "sample":
        return {"kind": kind, "rows": _log(rng, 1, 200), "vocab": _log(rng, 1000, 152064), "mix": rng.choice(["default", "mixed", "top-p"])}
    kv, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128])
    half = rng.choice(["bf16", "bf16", "f16"])
    if kind == "append":
        return {"kind": kind, "B": _log(rng, 1, 200), "heads": kv * rng.choice([1, 2, 4, 5]), "kv_heads": kv, "dim": dim, "half": half,
                "rot": rng.choice([dim, dim, dim // 2]), "far": _log(rng, 1, 131071), "norm": rng.random() < 0.5}
    B = _log(rng, 1, 48)
    # the batch's slots: no more than the largest listed case holds
    hi = min(_log(rng, 1, 131072), 460000 // B)
    lo = rng.randint(0, hi)
    if kind == "evict":
        hi = min(hi, 380000 // B, 32768)
        lo = min(lo, hi)
        budget = _log(rng, 1, max(1, hi))
        sink = rng.randint(0, min(4, budget))
        return {"kind": kind, "B": B, "lo": lo, "hi": hi, "kv_heads": kv, "dim": dim, "half": half, "budget": budget, "sink": sink,
                "window": rng.randint(0, budget - sink)}
    return {"kind": kind, "B": B, "lo": lo, "hi": hi, "heads": kv * rng.choice([1, 2, 4, 5, 8, 16] if kv <= 2 else [1, 2, 4, 5]), "kv_heads": kv,
            "dim": dim, "half": half, "window": rng.choice([0, 0, _log(rng, 1, 4096)]), "weights": rng.random() < 0.4}


def _lengths(c):
    n, lo, hi = c["B"], c["lo"], c["hi"]
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def work(c):
    if c["kind"] == "sample":
        return {"bytes": 4.0 * c["rows"] * c["vocab"], "flops": 0.0}
    n, d = c["kv_heads"], c["dim"]
    if c["kind"] == "append":
        return {"bytes": c["B"] * d * (4.0 * (c["heads"] + 2 * n) + 4.0 * c["heads"] + 4.0 * n), "flops": 6.0 * c["B"] * d * (c["heads"] + n)}
    lens = _lengths(c)
    if c["kind"] == "evict":
        kept = sum(min(x, c["budget"]) for x in lens)
        # every weight once; of what stays, keys and values (2 bytes), the weight and the position, read and written
        return {"bytes": n * (4.0 * sum(lens) + kept * (8.0 * d + 4.0 * 3)), "flops": 0.0}
    seen = sum(min(x, c["window"] or x) for x in lens)
    io = 8.0 * c["B"] * c["heads"] * d + (8.0 * n * sum(lens) if c["weights"] else 0.0)
    return {"bytes": 4.0 * n * d * seen + io, "flops": 4.0 * c["heads"] * d * seen}


# ------------------------------------------------------------------------------------------- inputs
def _half(c):
    return torch.bfloat16 if c["half"] == "bf16" else torch.float16


def _pool(c, pages, gen):
    shape = (pages, c["kv_heads"], PAGE, c["dim"])
    return [torch.randn(shape, device="cuda", generator=gen, dtype=_half(c)) for _ in range(2)]


def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rs = np.random.default_rng(seed)
    randn = lambda *shape: torch.randn(shape, device="cuda", generator=gen)  # noqa: E731
    rand = lambda *shape: torch.rand(shape, device="cuda", generator=gen)  # noqa: E731
    s = dict(c)
    if c["kind"] == "sample":
        R, V = c["rows"], c["vocab"]
        # a model's logits: a broad bulk and some dozens of candidates above it
        s["logits"] = randn(R, V) * 2.0
        at = torch.randint(0, V, (R, 64), device="cuda", generator=gen)
        s["logits"].scatter_(1, at, 6.0 + 8.0 * rand(R, 64))
        full = lambda x, t=torch.float32: torch.full((R,), x, device="cuda", dtype=t)  # noqa: E731
        s["temperature"], s["top_k"], s["top_p"], s["min_p"] = full(0.7), full(40, torch.int32), full(0.95), full(0.0)
        if c["mix"] == "top-p":
            s["temperature"], s["top_k"], s["top_p"] = full(1.0), full(0, torch.int32), 0.5 + 0.45 * rand(R)
        elif c["mix"] == "mixed":
            which = torch.arange(R, device="cuda") % 5
            s["temperature"] = torch.where(which == 0, torch.zeros_like(s["temperature"]), 0.5 + 0.7 * rand(R))
            s["top_k"] = torch.where(which == 1, torch.randint(1, 200, (R,), device="cuda", generator=gen), 0).to(torch.int32)
            s["top_p"] = torch.where((which == 1) | (which == 2), 0.8 + 0.19 * rand(R), full(1.0))
            s["min_p"] = torch.where(which == 3, 0.02 + 0.1 * rand(R), full(0.0))
        s["u"] = rand(R)
        s["tokens"], s["status"] = full(-1, torch.int32), full(-1, torch.int32)
        return s
    B, n, d = c["B"], c["kv_heads"], c["dim"]
    if c["kind"] == "append":
        lens = rs.integers(1, 3 * PAGE + 1, B)   # slots are few here (a budgeted cache), positions are not
        s["inv_freq"] = torch.tensor(1e6 ** (-np.arange(0, c["rot"], 2) / max(1, c["rot"])), dtype=torch.float32, device="cuda")
        s["positions"] = torch.tensor(rs.integers(0, c["far"] + 1, B), dtype=torch.int32, device="cuda")
        s["qkv"] = randn(B, (c["heads"] + 2 * n) * d)
        s["qn"], s["kn"] = (1.0 + 0.1 * randn(d), 1.0 + 0.1 * randn(d)) if c["norm"] else (None, None)
        s["q"] = torch.empty(B, c["heads"] * d, device="cuda")
    else:
        lens = rs.permutation(np.array(_lengths(c)))
    top = max(1, int(lens.max()))
    width = 3 if c["kind"] == "append" else -(-top // PAGE)
    used = -(-lens // PAGE)
    keep = -(-min(top, c["budget"]) // PAGE) if c["kind"] == "evict" else 0
    pages = 3 * B if c["kind"] == "append" else int(used.sum()) + B * keep
    order = rs.permutation(max(1, pages)).astype(np.int32)
    table = np.zeros((B, width), np.int32)
    starts = np.concatenate([[0], np.cumsum(used)])
    for b in range(B):
        table[b, :used[b]] = order[starts[b]:starts[b + 1]]
    s["k"], s["v"] = _pool(c, max(1, pages), gen)
    s["table"], s["len"], s["max_len"] = torch.tensor(table, device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda"), top
    if c["kind"] == "attend":
        s["q"], s["scale"] = 2.0 * randn(B, c["heads"] * d), d ** -0.5
        s["out"] = torch.empty(B, c["heads"] * d, device="cuda")
        s["weight_in"], s["weight"] = (rand(B, n, top), torch.zeros(B, n, top, device="cuda")) if c["weights"] else (None, None)
    if c["kind"] == "evict":
        room = min(top, c["budget"])
        s["weight"] = torch.empty(B, n, top, device="cuda").exponential_(1.0, generator=gen)
        s["position"] = torch.arange(top, dtype=torch.int32, device="cuda").expand(B, n, top).contiguous() * 3
        s["to_table"] = torch.tensor(order[starts[B]:starts[B] + B * keep].reshape(B, keep), device="cuda")
        s["to_len"] = torch.zeros(B, dtype=torch.int32, device="cuda")
        s["to_weight"] = torch.zeros(B, n, room, device="cuda")
        s["to_position"] = torch.zeros(B, n, room, dtype=torch.int32, device="cuda")
        s["room"] = room
    return s


# ------------------------------------------------------------------------------------------- plain forms
def _gather(pool, table, count):
    """Slots 0 .. count - 1 of every sequence, as [B][heads][count][dim] in 32 bits."""
    x = pool[table.long()].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])[:, :, :count].float()


def _plain_attend(s):
    B, H, n, d, top = s["B"], s["heads"], s["kv_heads"], s["dim"], s["max_len"]
    slot, ln = torch.arange(top, device="cuda"), s["len"].long()[:, None]
    seen = slot < ln
    if s["window"]:
        seen = seen & (slot >= ln - s["window"])
    k, v = _gather(s["k"], s["table"], top), _gather(s["v"], s["table"], top)
    q = (s["q"].view(B, n, H // n, d) * s["scale"]).transpose(2, 3).contiguous()
    score = torch.matmul(k, q).transpose(2, 3).contiguous()                 # [B][n][G][top]
    score = score.masked_fill(~seen[:, None, None, :], -math.inf)
    most = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(most == -math.inf, torch.zeros_like(most), most))
    total = e.sum(-1, keepdim=True)
    p = torch.where(total > 0, e / total, torch.zeros_like(e))
    s["out"].copy_(torch.matmul(p, v).view(B, H * d))
    if s["weight"] is None:
        return {"out": s["out"]}
    s["weight"].copy_(torch.where((slot < ln)[:, None, :], s["weight_in"] + p.sum(2), s["weight"]))
    return {"out": s["out"], "weight": s["weight"]}


def _plain_append(s):
    B, H, n, d, rot = s["B"], s["heads"], s["kv_heads"], s["dim"], s["rot"]
    x = s["qkv"].view(B, H + 2 * n, d)
    qk = x[:, :H + n]
    if s["qn"] is not None:
        w = torch.cat([s["qn"].expand(H, d), s["kn"].expand(n, d)])
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + 1e-6) * w
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()       # far positions: 32 bits lose the angle
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b = qk[..., :rot // 2], qk[..., rot // 2:rot]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin, qk[..., rot:]], -1)
    s["q"].copy_(qk[:, :H].reshape(B, H * d))
    at = s["len"].long() - 1
    page = s["table"].long().gather(1, (at // PAGE)[:, None])[:, 0]
    s["k"][page, :, at % PAGE] = qk[:, H:].to(s["k"].dtype)
    s["v"][page, :, at % PAGE] = x[:, H + n:].to(s["v"].dtype)
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _plain_evict(s):
    n, top, room = s["kv_heads"], s["max_len"], s["room"]
    slot, ln = torch.arange(top, device="cuda"), s["len"].long()[:, None]
    kept = ln.clamp(max=s["budget"])
    always = ((slot < s["sink"]) | (slot >= ln - s["window"])) & (slot < ln)
    w = s["weight"].masked_fill(always[:, None], math.inf).masked_fill((slot >= ln)[:, None], -math.inf)
    first = w.sort(dim=-1, descending=True, stable=True).indices[..., :room]    # heaviest first, the lower slot first among equals
    here = (torch.arange(room, device="cuda") < kept)[:, None]               # [B][1][room]
    at = first.masked_fill(~here, top).sort(dim=-1).values.clamp(max=top - 1)    # in slot order
    head = torch.arange(n, device="cuda")[:, None]
    page = s["table"].long()[:, None].expand(-1, n, -1).gather(2, at // PAGE)
    to = torch.arange(room, device="cuda")
    to_page = s["to_table"].long()[:, to // PAGE][:, None]
    s["k"][to_page, head, to % PAGE] = torch.where(here[..., None], s["k"][page, head, at % PAGE], s["k"][to_page, head, to % PAGE])
    s["v"][to_page, head, to % PAGE] = torch.where(here[..., None], s["v"][page, head, at % PAGE], s["v"][to_page, head, to % PAGE])
    s["to_weight"].copy_(torch.where(here, s["weight"].gather(2, at), s["to_weight"]))
    s["to_position"].copy_(torch.where(here, s["position"].gather(2, at), s["to_position"]))
    s["to_len"].copy_(kept[:, 0])
    return _evicted(s)


def _evicted(s):
    return {"k": s["k"], "v": s["v"], "len": s["to_len"], "weight": s["to_weight"], "position": s["to_position"]}


def _plain_sample(s):
    v, index = s["logits"].double().sort(dim=-1, descending=True, stable=True)   # 64 bits: draws lie next to borders
    V = v.shape[1]
    rank = torch.arange(V, device="cuda")
    t = s["temperature"].double()[:, None]
    w = torch.exp((v - v[:, :1]) / torch.where(t > 0.001, t, torch.ones_like(t)))
    k = torch.where(s["top_k"] > 0, s["top_k"].clamp(max=V), V).long()[:, None]
    run = torch.where(rank < k, w, torch.zeros_like(w)).cumsum(-1)
    low = (w >= s["min_p"].double()[:, None]).sum(-1, keepdim=True)
    p = s["top_p"].double()[:, None]
    cut = torch.where(p < 1, (run < p * run[:, -1:]).sum(-1, keepdim=True) + 1, V)
    end = torch.minimum(torch.minimum(k, low), cut).clamp(1, V)
    goal = s["u"].double()[:, None] * run.gather(1, end - 1)
    pick = torch.minimum((run < goal).sum(-1, keepdim=True), end - 1)
    pick = torch.where(t > 0.001, pick, torch.zeros_like(pick))
    s["tokens"].copy_(index.gather(1, pick)[:, 0])
    s["status"].zero_()
    return {"tokens": s["tokens"], "status": s["status"]}


# ------------------------------------------------------------------------------------------- the framework's calls
def _ptr(t):
    return None if t is None else t.data_ptr()


def _cache(mlxr, s, to=""):
    return mlxr.PagedKV(k=_ptr(s["k"]), v=_ptr(s["v"]), table=_ptr(s[to + "table"]), len=_ptr(s[to + "len"]),
                        weight=_ptr(s.get(to + "weight")), position=_ptr(s.get(to + "position")),
                        n_pages=s["k"].shape[0], table_stride=s[to + "table"].shape[1], slot_stride=s["room"] if to else s["max_len"],
                        max_len=s["room"] if to else s["max_len"], B=s["B"], nKV=s["kv_heads"], D=s["dim"], st=int(s["half"] == "f16"))


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

    if s["kind"] == "sample":
        call, args = lib.mlxr_k_sample_rows, (_ptr(s["logits"]), s["rows"], s["vocab"], s["vocab"], _ptr(s["temperature"]), _ptr(s["top_k"]),
                                              _ptr(s["top_p"]), _ptr(s["min_p"]), _ptr(s["u"]), _ptr(s["tokens"]), _ptr(s["status"]),
                                              *work(lib.mlxr_k_sample_rows_work(s["rows"], s["vocab"])), stream)
    else:
        kv = _cache(mlxr, s)
        ref = ctypes.byref(kv)
        if s["kind"] == "attend":
            call, args = lib.mlxr_k_paged_attention, (ref, _ptr(s["q"]), s["heads"] * s["dim"], s["heads"], s["window"], s["scale"], _ptr(s["out"]),
                                                      s["heads"] * s["dim"], _ptr(s["weight_in"]), 1.0,
                                                      *work(lib.mlxr_k_paged_attention_work(ref, s["heads"])), stream)
        elif s["kind"] == "append":
            call, args = lib.mlxr_k_paged_append, (ref, _ptr(s["qkv"]), s["qkv"].shape[1], _ptr(s["inv_freq"]), _ptr(s["qn"]), _ptr(s["kn"]),
                                                   s["heads"], s["rot"], 0, _ptr(s["positions"]), 1e-6, _ptr(s["q"]), s["heads"] * s["dim"], stream)
        else:
            to = _cache(mlxr, s, "to_")
            call, args = lib.mlxr_k_paged_evict, (ref, ctypes.byref(to), s["budget"], s["sink"], s["window"],
                                                  *work(lib.mlxr_k_paged_evict_work(ref, s["budget"])), stream)
            s["to"] = to
        s["kv"] = kv
    return lambda: mlxr.check(call(*args))


def run(s):
    kind = s["kind"]
    if own:
        if "call" not in s:
            s["call"] = _calls(s)
        s["call"]()
        if kind == "attend":
            return {"out": s["out"]} if s["weight"] is None else {"out": s["out"], "weight": s["weight"]}
        if kind == "append":
            return {"q": s["q"], "k": s["k"], "v": s["v"]}
        return _evicted(s) if kind == "evict" else {"tokens": s["tokens"], "status": s["status"]}
    return {"attend": _plain_attend, "append": _plain_append, "evict": _plain_evict, "sample": _plain_sample}[kind](s)


# ------------------------------------------------------------------------------------------- the definition in 64 bits
def _exact_attend(s):
    B, H, n, d = s["B"], s["heads"], s["kv_heads"], s["dim"]
    out = torch.zeros(B, H, d, dtype=torch.float64, device="cuda")
    weight = s["weight"].double() if s["weight"] is not None else None
    for b, count in enumerate(s["len"].tolist()):
        start = max(0, count - s["window"]) if s["window"] else 0
        if count == 0:
            continue
        pages = s["table"][b, :-(-count // PAGE)].long()
        for h in range(n):
            k = s["k"][pages, h].reshape(-1, d)[start:count].double()
            v = s["v"][pages, h].reshape(-1, d)[start:count].double()
            q = s["q"][b].view(n, H // n, d)[h].double()
            p = torch.softmax(k @ q.t().contiguous() * float(s["scale"]), 0)
            out[b, h * (H // n):(h + 1) * (H // n)] = p.t().contiguous() @ v
            if weight is not None:
                weight[b, h, :count] = s["weight_in"][b, h, :count].double()
                weight[b, h, start:count] += p.sum(1)
    found = {"out": out.view(B, H * d)}
    return found if weight is None else {**found, "weight": weight}


def _exact_append(s):
    B, H, n, d, rot = s["B"], s["heads"], s["kv_heads"], s["dim"], s["rot"]
    x = s["qkv"].cpu().double().numpy().reshape(B, H + 2 * n, d)
    heads = x[:, :H + n].copy()
    if s["qn"] is not None:
        heads /= np.sqrt((heads ** 2).mean(-1, keepdims=True) + 1e-6)
        heads[:, :H] *= s["qn"].cpu().double().numpy()
        heads[:, H:] *= s["kn"].cpu().double().numpy()
    z = heads[..., :rot // 2] + 1j * heads[..., rot // 2:rot]
    z = z * np.exp(1j * s["positions"].cpu().numpy()[:, None] * s["inv_freq"].cpu().double().numpy())[:, None]
    heads[..., :rot] = np.concatenate([z.real, z.imag], -1)
    k, v = s["k"].double(), s["v"].double()
    for b, count in enumerate(s["len"].tolist()):
        page, at = int(s["table"][b, (count - 1) // PAGE]), (count - 1) % PAGE
        k[page, :, at] = torch.from_numpy(heads[b, H:]).to(k.device)
        v[page, :, at] = torch.from_numpy(x[b, H + n:]).to(v.device)
    return {"q": torch.from_numpy(heads[:, :H].reshape(B, H * d)), "k": k, "v": v}


def _exact_evict(s):
    k, v = s["k"].clone(), s["v"].clone()
    weight, position, lens = s["to_weight"].double(), s["to_position"].clone(), s["to_len"].clone()
    for b, count in enumerate(s["len"].tolist()):
        kept = min(count, s["budget"])
        lens[b] = kept
        for h in range(s["kv_heads"]):
            w = s["weight"][b, h, :count].cpu().numpy()
            chosen = np.arange(count)
            if count > kept:
                middle = np.arange(s["sink"], count - s["window"])
                middle = middle[np.lexsort((middle, -w[middle].astype(np.float64)))][:kept - s["sink"] - s["window"]]
                chosen = np.sort(np.concatenate([np.arange(s["sink"]), middle, np.arange(count - s["window"], count)]))
            i = torch.from_numpy(chosen).to(k.device)
            page, to, j = s["table"][b].long()[i // PAGE], s["to_table"][b].long(), torch.arange(kept, device=k.device)
            k[to[j // PAGE], h, j % PAGE] = s["k"][page, h, i % PAGE]
            v[to[j // PAGE], h, j % PAGE] = s["v"][page, h, i % PAGE]
            weight[b, h, :kept] = s["weight"][b, h, i].double()
            position[b, h, :kept] = s["position"][b, h, i]
    return {"k": k.double(), "v": v.double(), "len": lens, "weight": weight, "position": position}


def _exact_sample(s):
    found = []
    for r in range(s["rows"]):
        v = s["logits"][r].cpu().numpy().astype(np.float64)
        t, k, p, low, u = (float(s[x][r]) for x in ("temperature", "top_k", "top_p", "min_p", "u"))
        order = np.lexsort((np.arange(len(v)), -v))
        if t <= 0.001:
            found.append(int(order[0]))
            continue
        if k > 0:
            order = order[:int(k)]
        w = np.exp((v[order] - v[order[0]]) / t)
        mass, end = math.fsum(w), len(w)
        run = np.cumsum(w)
        if p < 1:
            end = min(end, int(np.searchsorted(run, p * mass)) + 1)
        under = np.nonzero(w < low)[0]
        if under.size:
            end = min(end, int(under[0]))
        end = max(1, end)
        found.append(int(order[min(end - 1, int(np.searchsorted(run[:end], u * run[end - 1])))]))
    return {"tokens": torch.tensor(found, dtype=torch.int32), "status": torch.zeros(len(found), dtype=torch.int32)}


def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"] == "sample" and c["rows"] * c["vocab"] > 60_000_000:
        return None   # sorted on the host, row by row
    if c["kind"] == "evict" and c["kv_heads"] * sum(_lengths(c)) > 4_000_000:
        return None
    return {"attend": _exact_attend, "append": _exact_append, "evict": _exact_evict, "sample": _exact_sample}[c["kind"]](s)
