"""The operators around a layer's attention, as measured cases.

Four operators, each called as an attention layer of a serving step calls it:

- ``rotary``: rotary positions on the queries and keys of a step.
- ``norm_rotary``: the RMS norm of every query and key head, then the rotation.
- ``append``: the same on the way into a paged cache: rotated queries out, rotated keys and plain values into the
  pages that the step's slots name.
- ``shared``: decode rows whose leading keys lie in the same pages (a system prompt, a document, parallel samples of one
  prompt) attend them computed once for all, each row then its own keys.

Queries, keys and values are views of one fused projection output, as a layer has them. The rotary table (fp32 cosines,
then sines, a row for each position) is computed in 64 bits by ``prepare``: a program lays it out once and keeps it.
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

_PACKAGE = str(Path(__file__).resolve().parents[1] / "lean-vllm_amd")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
BASE = dict(op="rotary", heads=32, kv_heads=8, dim=128, dtype="bf16", lengths=0,
            # rotary, norm_rotary, append
            tokens=0, chunks=0, rotary_dim=128, interleaved=False, base=1000000.0, scaling="none", factor=1.0,
            trained=32768, max_position=40960, norm=False, page=256, layout="NHD", skip=0,
            # shared
            rows=0, queries=1, shared=0, own_lo=0, own_hi=0)


def listed():
    return [
        # One user's next token on a small model: the rotation alone, where latency counts.
        dict(BASE, name="rotary_token", heads=16, kv_heads=8, tokens=1, lengths=1),
        # A large token budget, prompt chunks and decoding rows, one layer's queries and keys.
        dict(BASE, name="rotary_budget", tokens=8192, chunks=4, lengths=2),
        # Interleaved pairs over half of each head, as some model families rotate, on an odd number of tokens.
        dict(BASE, name="rotary_partial", heads=40, dim=64, dtype="fp16", rotary_dim=32, interleaved=True, tokens=1531,
             chunks=3, base=10000.0, scaling="linear", factor=4.0, lengths=3),
        # A decode batch of a model that norms its heads.
        dict(BASE, name="norm_rotary_decode", op="norm_rotary", norm=True, tokens=96, lengths=4),
        # A long prompt's step with positions far past the trained ones.
        dict(BASE, name="norm_rotary_long", op="norm_rotary", norm=True, tokens=16384, chunks=2, scaling="yarn",
             factor=4.0, max_position=131072, lengths=5),
        # A handful of users on a small model, one token each, into the cache.
        dict(BASE, name="append_few", op="append", heads=16, kv_heads=8, norm=True, tokens=3, lengths=6),
        # The large token budget into small pages.
        dict(BASE, name="append_budget", op="append", norm=True, tokens=8192, chunks=4, page=16, lengths=7),
        # An ordinary prompt step of 64-wide heads into a head-major cache, some tokens of which are not stored.
        dict(BASE, name="append_ragged", op="append", heads=64, dim=64, rotary_dim=64, base=500000.0, scaling="llama3",
             factor=8.0, trained=8192, max_position=65536, tokens=997, chunks=5, page=64, layout="HND", skip=37,
             lengths=8),
        # A few rows behind a short system prompt, on small pages.
        dict(BASE, name="shared_few", op="shared", heads=16, kv_heads=8, rows=4, shared=2048, own_lo=1, own_hi=300,
             page=16, lengths=9),
        # An ordinary batch behind a long system prompt.
        dict(BASE, name="shared_batch", op="shared", rows=64, shared=8192, own_lo=16, own_hi=1024, lengths=10),
        # Drafted tokens on 64-wide heads and a head-major cache.
        dict(BASE, name="shared_drafts", op="shared", heads=64, dim=64, dtype="fp16", page=64, layout="HND", rows=23,
             queries=3, shared=16384, own_lo=3, own_hi=700, lengths=11),
        # Many questions to one long document.
        dict(BASE, name="shared_document", op="shared", rows=200, shared=32768, own_lo=64, own_hi=2048, lengths=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    top = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["rotary", "norm_rotary", "append", "shared", "shared"])
        c = dict(BASE, op=op, lengths=rng.randrange(1 << 20), dtype=rng.choice(["bf16", "bf16", "fp16"]),
                 page=rng.choice([16, 16, 32, 48, 64, 256]), layout=rng.choice(["NHD", "NHD", "HND"]))
        c["heads"], c["kv_heads"] = rng.choice([(16, 8), (32, 8), (32, 8), (64, 8), (40, 8), (16, 2), (7, 1), (8, 8)])
        if op == "shared":
            c["dim"] = rng.choice([64, 128, 128])
            c["rotary_dim"] = c["dim"]
            c["queries"] = rng.choice([1, 1, 1, 2, 3, 5])
            c["rows"] = _log_int(rng, 1, 256)
            c["shared"] = c["page"] * max(1, _log_int(rng, 64, 65536) // c["page"])
            c["own_hi"] = max(c["queries"], _log_int(rng, 4, 4096))
            c["own_lo"] = max(c["queries"], c["own_hi"] // rng.choice([1, 4, 100]))
        else:
            c["dim"] = rng.choice([64, 128, 128, 80, 96, 256])
            c["interleaved"] = rng.random() < 0.4
            parts = [c["dim"], c["dim"], c["dim"] // 2 // 16 * 16, c["dim"] // 4 // 2 * 2]
            c["rotary_dim"] = rng.choice(parts)
            c["tokens"] = _log_int(rng, 1, 16384)
            c["chunks"] = rng.choice([0, 1, 2, 5]) if c["tokens"] >= 64 else 0
            c["base"] = rng.choice([10000.0, 500000.0, 1000000.0])
            c["scaling"] = rng.choice(["none", "linear", "ntk", "llama3", "yarn"])
            c["factor"] = 1.0 if c["scaling"] == "none" else rng.choice([2.0, 4.0, 8.0])
            c["trained"] = rng.choice([4096, 8192, 32768])
            c["max_position"] = rng.choice([40960, 65536, 131072])
            c["norm"] = op == "norm_rotary" or (op == "append" and rng.random() < 0.5)
            if op == "append":
                c["skip"] = rng.choice([0, 0, c["tokens"] // 16])
        if _cost(c) <= top and _tokens_fit(c):
            return c


def _tokens_fit(c):
    return c["op"] == "shared" or c["tokens"] * (c["heads"] + 2 * c["kv_heads"]) * c["dim"] <= 1 << 27


def _cost(c):
    w = work(c)
    return w["bytes"] / 5e12 + w["flops"] / 1e15


# ---------------------------------------------------------------------------------------------------------------
# Rows and work


def _own_lens(c):
    """Keys of every row behind the shared ones, its queries' own among them."""
    rng = np.random.default_rng(c["lengths"])
    return rng.integers(c["own_lo"], c["own_hi"] + 1, size=c["rows"])


def work(c):
    e = 2
    if c["op"] == "shared":
        lens, q, g = _own_lens(c), c["queries"], c["heads"] * c["dim"]
        tokens = c["rows"] * q
        keys = c["shared"] + int(lens.sum())
        seen = tokens * c["shared"] + int(sum(q * int(n) - q * (q - 1) // 2 for n in lens))
        return {"bytes": keys * 2 * c["kv_heads"] * c["dim"] * e + 2 * tokens * g * e, "flops": 4 * g * seen}
    t, d = c["tokens"], c["dim"]
    moved = c["heads"] + c["kv_heads"]  # heads read and written
    read = moved + (c["kv_heads"] if c["op"] == "append" else 0)
    written = c["tokens"] * moved * d
    if c["op"] == "append":
        written = t * c["heads"] * d + (t - c["skip"]) * 2 * c["kv_heads"] * d
    per_token = 8 + 4 * c["rotary_dim"] + (4 if c["op"] == "append" else 0)  # position, table row, slot
    flops = t * moved * (3 * c["rotary_dim"] + (4 * d if c["norm"] else 0))
    return {"bytes": (t * read * d + written) * e + t * per_token, "flops": flops}


# ---------------------------------------------------------------------------------------------------------------
# Inputs


def _frequencies(c):
    """Angle per position of every pair (64 bits), and the factor on cosines and sines."""
    r, base, f = c["rotary_dim"], c["base"], c["factor"]
    inv = base ** -(np.arange(0, r, 2, dtype=np.float64) / r)
    if c["scaling"] == "linear":
        return inv / f, 1.0
    if c["scaling"] == "ntk":
        return (base * f ** (r / max(r - 2, 1))) ** -(np.arange(0, r, 2, dtype=np.float64) / r), 1.0
    if c["scaling"] == "llama3":
        turns = c["trained"] * inv / (2 * math.pi)
        keep = np.clip((turns - 1.0) / (4.0 - 1.0), 0.0, 1.0)
        return inv * (keep + (1 - keep) / f), 1.0
    if c["scaling"] == "yarn":
        at = lambda turns: r * math.log(c["trained"] / (2 * math.pi * turns)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), r - 1)
        ramp = np.clip((np.arange(r // 2) - lo) / max(hi - lo, 1e-3), 0.0, 1.0)
        return inv * (1 - ramp + ramp / f), 0.1 * math.log(f) + 1.0
    return inv, 1.0


def _positions(c):
    """A step's positions: decoding rows anywhere, then chunks of consecutive ones."""
    rng = np.random.default_rng(c["lengths"])
    t, most = c["tokens"], c["max_position"]
    in_chunks = t - t // 64 if c["chunks"] else 0
    parts = [rng.integers(0, most, size=t - in_chunks)]
    cuts = np.sort(rng.integers(0, in_chunks + 1, size=max(c["chunks"] - 1, 0)))
    for n in np.diff([0, *cuts, in_chunks]):
        parts.append(np.arange(n) + rng.integers(0, most - n + 1))
    return np.concatenate(parts)[:t].astype(np.int64)


def _cache(c, blocks, gen):
    shape = (blocks, c["page"], c["kv_heads"], c["dim"])
    if c["layout"] == "HND":
        shape = (blocks, c["kv_heads"], c["page"], c["dim"])
    x = torch.randn(shape, device="cuda", dtype=torch.float32, generator=gen).to(DTYPES[c["dtype"]])
    return x.transpose(1, 2) if c["layout"] == "HND" else x


def prepare(case, seed):
    c, dt = case, DTYPES[case["dtype"]]
    rng = np.random.default_rng([seed, c["lengths"]])
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    h, hk, d = c["heads"], c["kv_heads"], c["dim"]
    if c["op"] == "shared":
        lens = _own_lens(c)
        tokens, page = c["rows"] * c["queries"], c["page"]
        head = c["shared"] // page
        tails = [-(-int(n) // page) for n in lens]
        blocks = head + sum(tails) + 3
        perm = rng.permutation(blocks).astype(np.int32)
        tables = np.full((c["rows"], head + max(tails)), -1, np.int32)
        tables[:, :head] = perm[:head]
        at = head
        for i, n in enumerate(tails):
            tables[i, head:head + n] = perm[at:at + n]
            at += n
        s["q"] = (2 * torch.randn(tokens, h, d, device="cuda", generator=gen)).to(dt)
        s["k_cache"], s["v_cache"] = _cache(c, blocks, gen), _cache(c, blocks, gen)
        s["tables"] = torch.from_numpy(tables).cuda()
        s["lens"] = torch.from_numpy((c["shared"] + lens).astype(np.int32)).cuda()
        return s
    t = c["tokens"]
    s["positions"] = torch.from_numpy(_positions(c)).cuda()
    inv, amp = _frequencies(c)
    angles = torch.arange(c["max_position"], device="cuda", dtype=torch.float64)[:, None] * torch.from_numpy(inv).cuda()
    s["table"] = torch.cat((angles.cos() * amp, angles.sin() * amp), 1).float()
    qkv = torch.randn(t, (h + 2 * hk) * d, device="cuda", generator=gen)
    qkv *= 0.5 + torch.rand(d, device="cuda", generator=gen).repeat(h + 2 * hk)  # channels of unlike sizes
    qkv = qkv.to(dt)
    q, k, v = qkv.split((h * d, hk * d, hk * d), 1)
    s["q"], s["k"], s["v"] = q.view(t, h, d), k.view(t, hk, d), v.view(t, hk, d)
    if c["norm"]:
        s["q_weight"], s["k_weight"] = ((1 + 0.3 * torch.randn(d, device="cuda", generator=gen)).to(dt)
                                        for _ in range(2))
    if c["op"] == "append":
        blocks = t // c["page"] + 9
        s["k_cache"], s["v_cache"] = _cache(c, blocks, gen), _cache(c, blocks, gen)
        slots = np.arange(t) + rng.integers(0, blocks * c["page"] - t + 1)  # consecutive, then over scattered pages
        slots = rng.permutation(blocks)[slots // c["page"]] * c["page"] + slots % c["page"]
        slots[rng.permutation(t)[:c["skip"]]] = -1
        s["slots"] = torch.from_numpy(slots.astype(np.int32)).cuda()
        s["stored"] = torch.from_numpy(np.flatnonzero(slots >= 0)).cuda()  # the tokens that have a slot, a host's list
    return s


# ---------------------------------------------------------------------------------------------------------------
# One pass


def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    return _plain_shared(s, c) if c["op"] == "shared" else _plain_rotary(s, c)


def _run_own(s, c):
    import lvattn

    if c["op"] == "rotary":
        return lvattn.apply_rotary(s["q"], s["k"], s["positions"], s["table"], interleaved=c["interleaved"])
    if c["op"] == "norm_rotary":
        return lvattn.norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["table"], eps=EPS,
                                  interleaved=c["interleaved"])
    backend = lvattn.MI355XAttention(c["heads"], c["dim"], c["dim"] ** -0.5, c["kv_heads"])
    if c["op"] == "append":
        q = backend.append_kvcache(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], s["positions"],
                                   s["table"], q_weight=s.get("q_weight"), k_weight=s.get("k_weight"), eps=EPS,
                                   interleaved=c["interleaved"])
        return q, s["k_cache"], s["v_cache"]
    context = lvattn.Context(context_lens=s["lens"], block_tables=s["tables"])
    return backend.decode_shared(s["q"], s["k_cache"], s["v_cache"], context, c["shared"])


def _rotate(x, cos, sin, interleaved):
    """fp32 ``x`` [T, H, D]; ``cos``, ``sin`` [T, 1, r / 2]."""
    half = cos.size(-1)
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, x[..., 2 * half:]), -1)


def _plain_rotary(s, c):
    row = s["table"][s["positions"]][:, None]
    cos, sin = row.chunk(2, -1)
    q, k = s["q"].float(), s["k"].float()
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_weight"].float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_weight"].float()
    dt = s["q"].dtype
    q, k = _rotate(q, cos, sin, c["interleaved"]).to(dt), _rotate(k, cos, sin, c["interleaved"]).to(dt)
    if c["op"] != "append":
        return q, k
    slots = s["slots"][s["stored"]].long()
    page, at = slots // c["page"], slots % c["page"]
    s["k_cache"][page, at] = k[s["stored"]]
    s["v_cache"][page, at] = s["v"][s["stored"]]
    return q, s["k_cache"], s["v_cache"]


def _plain_shared(s, c):
    rows, n, hk, d = c["rows"], c["queries"], c["kv_heads"], c["dim"]
    g, shared, head = c["heads"] // hk, c["shared"], c["shared"] // c["page"]
    q = s["q"].float().mul(d ** -0.5).view(rows, n, hk, g, d)
    # The prefix once for all: [hk, rows n g, d] against [hk, shared, d].
    first = s["tables"][0, :head].long()
    kp = s["k_cache"][first].float().reshape(shared, hk, d).permute(1, 2, 0)
    vp = s["v_cache"][first].float().reshape(shared, hk, d).transpose(0, 1)
    sp = (q.permute(2, 0, 1, 3, 4).reshape(hk, rows * n * g, d) @ kp).view(hk, rows, n, g, shared)
    # Each row's own keys, padded to the longest row's.
    tail = s["tables"][:, head:].long().clamp(min=0)
    width = tail.size(1) * c["page"]
    ko = s["k_cache"][tail].float().reshape(rows, width, hk, d).permute(0, 2, 3, 1)
    vo = s["v_cache"][tail].float().reshape(rows, width, hk, d).transpose(1, 2)
    so = (q.permute(0, 2, 1, 3, 4).reshape(rows, hk, n * g, d) @ ko).view(rows, hk, n, g, width)
    sees = s["lens"].long()[:, None] - shared - n + 1 + torch.arange(n, device="cuda")  # keys of its own each query sees
    hidden = torch.arange(width, device="cuda") >= sees[..., None]
    so = so.masked_fill(hidden[:, None, :, None], -math.inf).transpose(0, 1)
    most = torch.maximum(sp.amax(-1), so.amax(-1))[..., None]
    sp, so = (sp - most).exp(), (so - most).exp()
    total = (sp.sum(-1) + so.sum(-1))[..., None]
    op = (sp.reshape(hk, rows * n * g, shared) @ vp).view(hk, rows, n, g, d)
    oo = (so.transpose(0, 1).reshape(rows, hk, n * g, width) @ vo).view(rows, hk, n, g, d).transpose(0, 1)
    return ((op + oo) / total).permute(1, 2, 0, 3, 4).reshape(rows * n, hk * g, d).to(s["q"].dtype)


# ---------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits


def exact(case, seed):
    c, s = case, prepare(case, seed)
    return _exact_shared(s, c) if c["op"] == "shared" else _exact_rotary(s, c)


def _exact_rotary(s, c):
    inv, amp = _frequencies(c)
    angle = s["positions"].double()[:, None, None] * torch.from_numpy(inv).cuda()
    turn = torch.polar(torch.full_like(angle, amp), angle)  # a pair of dims is a complex number, turned

    def rotated(x, weight):
        x = x.double()
        if c["norm"]:
            x = x / (x.pow(2).sum(-1, keepdim=True) / c["dim"] + EPS).sqrt() * weight.double()
        r = c["rotary_dim"]
        pairs = x[..., :r].unflatten(-1, (r // 2, 2) if c["interleaved"] else (2, r // 2))
        if not c["interleaved"]:
            pairs = pairs.transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        y = y.flatten(-2) if c["interleaved"] else y.transpose(-1, -2).flatten(-2)
        return torch.cat((y, x[..., r:]), -1)

    q, k = rotated(s["q"], s.get("q_weight")), rotated(s["k"], s.get("k_weight"))
    if c["op"] != "append":
        return q, k
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    slots = s["slots"].long()
    kept = slots >= 0
    page, at = slots[kept] // c["page"], slots[kept] % c["page"]
    k_cache[page, at] = k[kept]
    v_cache[page, at] = s["v"].double()[kept]
    return q, k_cache, v_cache


def _exact_shared(s, c):
    hk, d, n = c["kv_heads"], c["dim"], c["queries"]
    g, shared, page = c["heads"] // hk, c["shared"], c["page"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    tables, lens = s["tables"].long(), s["lens"].tolist()
    first = tables[0, :shared // page]
    kp, vp = (x[first].reshape(shared, hk, d).double() for x in (s["k_cache"], s["v_cache"]))
    for i, length in enumerate(lens):
        rest = tables[i, shared // page:-(-length // page)]
        ko, vo = (x[rest].reshape(-1, hk, d)[:length - shared].double() for x in (s["k_cache"], s["v_cache"]))
        q = s["q"][i * n:(i + 1) * n].double().view(n, hk, g, d)
        for h in range(hk):
            k, v = torch.cat((kp[:, h], ko[:, h])), torch.cat((vp[:, h], vo[:, h]))
            scores = q[:, h].reshape(n * g, d) @ k.T * d ** -0.5
            last = torch.arange(n, device="cuda").repeat_interleave(g) + length - n
            scores = scores.masked_fill(torch.arange(length, device="cuda") > last[:, None], -math.inf)
            out[i * n:(i + 1) * n].view(n, hk, g, d)[:, h] = (scores.softmax(-1) @ v).view(n, g, d)
    return out
