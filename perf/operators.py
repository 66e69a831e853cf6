"""Measured cases of the attention operators over a paged key-value cache: appending the new tokens' keys and values
(rotated on the way), and attention of the new tokens -- one per sequence while decoding, a few while drafted tokens are
checked, many while a prompt is read -- over what the cache holds.

The operands are the ones a decoder layer has in hand: the fused q|k|v product's f32 result [tokens, (heads + 2 kv heads) *
dim], of which q, k and v are column slices; the layer's cache, two 16-bit tensors [pages, kv heads, page, dim]; and for
the batch a page table, the sequences' lengths (new tokens included) and, unless every sequence has exactly one new token,
the first token row of each sequence.  Token j of a sequence with n new tokens and length L sits at position L - n + j and
sees the keys up to its own position (at most `window` of them where a window is set).

`own` selects between the framework's operators and the same mathematics in elementary torch operations.
"""
import math
import random

import torch

own = False

ROPE_BASE = 1.0e6
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _case(name, op, seqs, new, lens, heads, kv_heads, dim, page, cache, out="f32", rope="halves", rotary=None, window=0):
    return {"name": name, "op": op, "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "len_lo": lens[0], "len_hi": lens[1],
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "cache": cache, "out": out, "rope": rope,
            "rotary": dim if rotary is None else rotary, "window": window}


def listed():
    return [
        # one user's next token: the smallest append, all launch latency (the 27B-class layer's heads: 40 over 8 of 128)
        _case("append 1 token", "append", 1, (1, 1), (1001, 1001), 40, 8, 128, 64, "bf16"),
        # a full decode batch, far positions, small pages, adjacent-pair rotation
        _case("append 64 tokens", "append", 64, (1, 1), (517, 120011), 32, 8, 128, 16, "f16", rope="pairs"),
        # several prompts of odd lengths admitted together, wide heads of which a quarter is rotated
        _case("append ragged prompts", "append", 5, (311, 1403), (311, 5000), 16, 4, 256, 32, "bf16", rotary=64),
        # one long prompt
        _case("append 16384 tokens", "append", 1, (16384, 16384), (16384, 16384), 40, 8, 128, 64, "bf16"),
        # one user, a short conversation: latency again
        _case("decode 1 x 100", "attend", 1, (1, 1), (100, 100), 40, 8, 128, 64, "bf16"),
        # one user, a book in the context: few rows, a very long cache
        _case("decode 1 x 131000", "attend", 1, (1, 1), (131000, 131000), 40, 8, 128, 64, "bf16"),
        # a full serving batch of uneven conversations, small pages
        _case("decode 64 x 0.7k-8k", "attend", 64, (1, 1), (700, 8190), 40, 8, 128, 16, "f16"),
        # wide heads, a sliding window, a quarter rotated
        _case("decode 24 x window 4096", "attend", 24, (1, 1), (300, 9000), 16, 2, 256, 32, "bf16", rotary=64, window=4096),
        # drafted tokens checked in one go: five new tokens per sequence
        _case("draft 8 x 5", "attend", 8, (5, 5), (1200, 4100), 40, 8, 64, 64, "f16", rope="pairs"),
        # one prompt read at once, the result in the prefill product's activation type
        _case("prompt 4096", "attend", 1, (4096, 4096), (4096, 4096), 40, 8, 128, 64, "bf16", out="bf16"),
        # chunks of three prompts on top of what the cache already holds of them
        _case("prompt chunks", "attend", 3, (350, 1001), (2000, 9001), 32, 4, 128, 32, "f16", out="bf16"),
        # a layer's whole mixer for a decode step: append, then attend
        _case("step 8 x 4k", "step", 8, (1, 1), (3900, 4200), 40, 8, 128, 64, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "append", "decode", "decode", "decode", "draft", "prompt", "prompt", "step"])
    dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    page, cache = rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "f16"])
    kw = {"rope": rng.choice(["halves", "pairs"]), "rotary": rng.choice([dim, dim, dim // 4])}
    if op == "append":
        if rng.random() < 0.5:
            n = (1, 1)
            seqs = _log_int(rng, 1, 128)
        else:
            seqs = rng.randint(1, 6)
            hi = _log_int(rng, 8, 16384 // seqs)
            n = (max(1, hi // 3), hi)
        hi = n[1] + _log_int(rng, 1, 4000)
        return _case("", "append", seqs, n, (n[1], hi), heads, kv_heads, dim, page, cache, **kw)
    if op in ("decode", "step", "draft"):
        new = 1 if op != "draft" else rng.randint(2, 8)
        seqs = _log_int(rng, 1, 64)
        # at most about the keys of the largest listed decode batch, and at most the longest listed context
        most = min(131000, 64 * 4400 * 8 * 128 // (seqs * kv_heads * dim))
        hi = _log_int(rng, 16, most)
        lo = max(new, hi // rng.choice([1, 2, 10]))
        window = rng.choice([0, 0, 0, 128, 1000])
        return _case("", "step" if op == "step" else "attend", seqs, (new, new), (lo, max(lo, hi)), heads, kv_heads, dim, page, cache,
                     out="f32" if op != "draft" else rng.choice(["f32", "bf16"]), window=window, **kw)
    seqs = rng.randint(1, 4)
    new = _log_int(rng, 16, 4096 // seqs)
    # query-key pairs times width: at most the listed prompts'
    while seqs * heads * dim * new * new > 40 * 128 * 4096 * 4096:
        new = new * 3 // 4
    hi = min(_log_int(rng, new, 16384), max(new, 20 * 128 * 4096 * 4096 // (seqs * heads * dim * new)))
    return _case("", "attend", seqs, (max(1, new // 2), new), (new, max(new, hi)), heads, kv_heads, dim, page, cache,
                 out=rng.choice(["bf16", "bf16", "f32"]) if new <= 1024 else "bf16", window=rng.choice([0, 0, 500]), **kw)


def _spread(n, lo, hi, phase):
    """n whole numbers over [lo, hi], uneven but fixed by the case."""
    if n == 1:
        return [hi]
    return [lo + int((hi - lo) * ((phase + 0.6180339887 * i) % 1.0) + 0.5) for i in range(n)]


def _counts(case):
    """Per sequence: its new tokens and its length (new tokens included)."""
    new = _spread(case["seqs"], case["new_lo"], case["new_hi"], 0.35)
    lens = [max(a, b) for a, b in zip(new, _spread(case["seqs"], case["len_lo"], case["len_hi"], 0.9))]
    return new, lens


def _inputs(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    new, lens = _counts(case)
    S, H, HK, D, P = case["seqs"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    cols = max((n + P - 1) // P for n in lens) + 2
    used = [(n + P - 1) // P for n in lens]
    n_pages = sum(used) + 3
    perm = random.Random(seed).sample(range(n_pages), n_pages)
    table = torch.full((S, cols), -1, dtype=torch.int32)
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = torch.tensor(perm[at:at + u], dtype=torch.int32)
        at += u
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    ty = _TYPES[case["cache"]]
    shape = (n_pages, HK, P, D)
    qkv = torch.randn((starts[-1], (H + 2 * HK) * D), generator=g, device=dev)
    qkv[:, :H * D] *= 1.5
    return {"qkv": qkv, "k_cache": torch.randn(shape, generator=g, device=dev).to(ty),
            "v_cache": torch.randn(shape, generator=g, device=dev).to(ty), "table": table.to(dev),
            "lens": torch.tensor(lens, dtype=torch.int32, device=dev), "starts": torch.tensor(starts, dtype=torch.int32, device=dev),
            "new_max": max(new), "len_max": max(lens), "one_each": max(new) == 1}


_kept = {}


def _context():
    """The program's context, made once."""
    import ferric_b200 as F

    if "ctx" not in _kept:
        _kept["ctx"] = F.Context(torch.cuda.current_device())
    return _kept["ctx"]


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    H, HK, D = case["heads"], case["kv_heads"], case["dim"]
    s["q"], s["k"], s["v"] = s["qkv"][:, :H * D], s["qkv"][:, H * D:(H + HK) * D], s["qkv"][:, (H + HK) * D:]
    s["freq"] = ROPE_BASE ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64, device="cuda") / case["rotary"])
    if own:
        import ferric_b200 as F

        ctx = _context()
        s["rope"] = F.Rope(ctx, case["rotary"], base=ROPE_BASE, interleaved=case["rope"] == "pairs")
        s["cache"] = F.KVCache(ctx, s["k_cache"], s["v_cache"])
        s["seqs"] = F.KVSeqs(s["table"], s["lens"], None if s["one_each"] else s["starts"])
    return s


# ---- the plain forms ------------------------------------------------------------------------------
def _positions(s):
    """Per token row: its sequence, its index among the sequence's new tokens and its position."""
    rows = torch.arange(s["qkv"].shape[0], device="cuda")
    seq = torch.searchsorted(s["starts"][1:].long(), rows, right=True)
    j = rows - s["starts"].long()[seq]
    n = (s["starts"][1:] - s["starts"][:-1]).long()[seq]
    return seq, j, s["lens"].long()[seq] - n + j


def _rotate(s, x, pos):
    """x[tokens, heads, dim] with its first `rotary` elements turned by position * frequency (angles in 64 bits)."""
    c = s["case"]
    ang = pos.double()[:, None] * s["freq"]
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]
    r = c["rotary"]
    if c["rope"] == "pairs":
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y, x[..., r:]], -1)


def _append(s):
    c = s["case"]
    seq, _, pos = _positions(s)
    page = s["table"].long()[seq, pos // c["page"]]
    slot = pos % c["page"]
    s["k_cache"][page, :, slot] = _rotate(s, s["k"].unflatten(1, (c["kv_heads"], c["dim"])), pos).to(s["k_cache"].dtype)
    s["v_cache"][page, :, slot] = s["v"].unflatten(1, (c["kv_heads"], c["dim"])).to(s["v_cache"].dtype)
    return s["k_cache"], s["v_cache"]


def _attend(s):
    c = s["case"]
    S, H, HK, D, n, L = c["seqs"], c["heads"], c["kv_heads"], c["dim"], s["new_max"], s["len_max"]
    seq, j, pos = _positions(s)
    q = torch.zeros((S, n, H, D), device="cuda")
    q[seq, j] = _rotate(s, s["q"].unflatten(1, (H, D)), pos) * (1.0 / math.sqrt(D))
    q = q.unflatten(2, (HK, H // HK)).permute(0, 2, 1, 3, 4).flatten(2, 3)                 # [S, HK, n * group, D]
    pages = s["table"][:, :(L + c["page"] - 1) // c["page"]].long().clamp(min=0)
    k = s["k_cache"][pages].transpose(1, 2).flatten(2, 3)[:, :, :L].float()                # [S, HK, L, D]
    w = q @ k.transpose(2, 3)
    del k
    w = w.unflatten(2, (n, H // HK))
    key = torch.arange(L, device="cuda")
    row = s["lens"].long()[:, None] - (s["starts"][1:] - s["starts"][:-1]).long()[:, None] + torch.arange(n, device="cuda")
    seen = key <= row[..., None]                                                           # [S, n, L]
    if c["window"]:
        seen &= key > row[..., None] - c["window"]
    w.masked_fill_(~seen[:, None, :, None], float("-inf"))
    w -= w.amax(-1, keepdim=True).clamp(min=-3.0e38)
    w = w.exp_().flatten(2, 3)
    total = w.sum(-1, keepdim=True)
    v = s["v_cache"][pages].transpose(1, 2).flatten(2, 3)[:, :, :L].float()
    o = (w @ v) / total.clamp(min=1e-30)
    o = o.unflatten(2, (n, H // HK)).permute(0, 2, 1, 3, 4).flatten(2, 4)                  # [S, n, H * D]
    return o[seq, j].to(_TYPES[c["out"]])


# ---- one pass ---------------------------------------------------------------------------------------
def _run_own(s):
    c = s["case"]
    out = {}
    if c["op"] in ("append", "step"):
        s["cache"].append(s["seqs"], s["k"], s["v"], rope=s["rope"])
        out["k"], out["v"] = s["k_cache"], s["v_cache"]
    if c["op"] in ("attend", "step"):
        out["o"] = s["cache"].attend(s["seqs"], s["q"], rope=s["rope"], window=c["window"], out_dtype=_TYPES[c["out"]])
    return out


def run(state):
    if own:
        return _run_own(state)
    out = {}
    if state["case"]["op"] in ("append", "step"):
        out["k"], out["v"] = _append(state)
    if state["case"]["op"] in ("attend", "step"):
        out["o"] = _attend(state)
    return out


def work(case):
    new, lens = _counts(case)
    H, HK, D = case["heads"], case["kv_heads"], case["dim"]
    tokens = sum(new)
    b = f = 0
    meta = 4 * (2 * case["seqs"] + 1 + sum(-(-n // case["page"]) for n in lens))
    if case["op"] in ("append", "step"):
        b += tokens * 2 * HK * D * (4 + 2)
        f += tokens * HK * case["rotary"] * 3
    if case["op"] in ("attend", "step"):
        w = case["window"]
        span = lambda n, x: x if not w else min(x, w + n - 1)              # keys that any of the sequence's new tokens sees
        pairs = 0
        for n, x in zip(new, lens):
            first, last = x - n + 1, x                                     # keys the first and the last new token see
            if not w or last <= w:
                pairs += (first + last) * n // 2
            else:
                grow = max(0, w - first)                                   # tokens that see fewer than `w` keys
                pairs += (first + w - 1) * grow // 2 + (n - grow) * w
        b += tokens * H * D * (4 + (4 if case["out"] == "f32" else 2)) + sum(span(n, x) for n, x in zip(new, lens)) * 2 * HK * D * 2
        f += 4 * D * H * pairs + tokens * H * case["rotary"] * 3
    return {"bytes": b + meta, "flops": f}


# ---- the definition in 64 bits, sequence by sequence --------------------------------------------------
def _turned(case, x, pos):
    """The rotation as a product of complex numbers."""
    r = case["rotary"]
    i = torch.arange(r // 2, dtype=torch.float64, device=x.device)
    ang = pos.double()[:, None] * torch.exp(-2.0 * i / r * math.log(ROPE_BASE))
    unit = torch.polar(torch.ones_like(ang), ang)[:, None]
    x = x.clone()
    if case["rope"] == "pairs":
        z = torch.complex(x[..., 0:r:2].contiguous(), x[..., 1:r:2].contiguous()) * unit
        x[..., 0:r:2], x[..., 1:r:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * unit
        x[..., :r // 2], x[..., r // 2:r] = z.real, z.imag
    return x


def exact(case, seed):
    s = _inputs(case, seed)
    new, lens = _counts(case)
    S, H, HK, D, P = case["seqs"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    kc, vc = s["k_cache"], s["v_cache"]
    out = {}
    if case["op"] in ("append", "step"):
        kx, vx = kc.double(), vc.double()
    o = torch.zeros((sum(new), H * D), dtype=torch.float64, device="cuda")
    at = 0
    for i in range(S):
        n, x = new[i], lens[i]
        pos = torch.arange(x - n, x, device="cuda")
        rows = s["qkv"][at:at + n].double()
        pages = s["table"][i, :(x + P - 1) // P].long()
        if case["op"] in ("append", "step"):
            kn = _turned(case, rows[:, H * D:(H + HK) * D].reshape(n, HK, D), pos)
            vn = rows[:, (H + HK) * D:].reshape(n, HK, D)
            kx[pages[pos // P], :, pos % P] = kn
            vx[pages[pos // P], :, pos % P] = vn
            # the cache holds the rounded values, and the attention reads those
            kc[pages[pos // P], :, pos % P] = kn.to(kc.dtype)
            vc[pages[pos // P], :, pos % P] = vn.to(vc.dtype)
        if case["op"] in ("attend", "step"):
            q = _turned(case, rows[:, :H * D].reshape(n, H, D), pos)
            key = torch.arange(x, device="cuda")[None]
            hidden = (key > pos[:, None]) | ((key <= pos[:, None] - case["window"]) if case["window"] else torch.zeros_like(key, dtype=torch.bool))
            for h in range(HK):
                kh = kc[pages, h].reshape(-1, D)[:x].double()
                vh = vc[pages, h].reshape(-1, D)[:x].double()
                for m in range(h * (H // HK), (h + 1) * (H // HK)):
                    z = (q[:, m] @ kh.T / math.sqrt(D)).masked_fill(hidden, -math.inf)
                    o[at:at + n, m * D:(m + 1) * D] = torch.softmax(z, -1) @ vh
        at += n
    if case["op"] in ("append", "step"):
        out["k"], out["v"] = kx, vx
    if case["op"] in ("attend", "step"):
        out["o"] = o
    return out
