"""Operators for several texts at once as a program calls them through g2hip, beside their plain form in torch.

Four kinds of case:
  prompt   causal attention over whole prompts of different lengths, packed one behind the other (grouped heads, fp32 or
           fp16 rows, keys that were there before)
  append   rows of keys and values appended to the 4-bit K/V cache, then the positions that they went to read back
  attend   single-query attention over that cache, one or many sequences, beams that share positions
  beam     a step of beam search: the best continuations of every group of beams, then the beams' ids and the table
           that says where their cached positions are, reordered

Sizes are the GPT-2 configurations' (12 to 25 heads of 64 dims, vocabulary 50257, context 1024), ragged ones in
between, and longer caches and prompts.  Activations, keys and values are N(0, 1).  Device buffers are torch tensors
given to the library as pointers.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
VOCAB, CTX, DH = 50257, 1024, 64
SCALE = 0.125
TILE = 32  # positions of the 4-bit cache that stand together
TILE_BYTES = 2 * TILE * DH // 2 + 2 * TILE * 2 * 2  # codes and bf16 scales (of 32 dims each) of keys and values
SPLITS = 32  # most parts of a head's positions in a call: the attention's workspace is (2 + 64) floats for each
SLACK = 5  # rows of a packed buffer behind the last sequence
INF = float("inf")


def listed():
    return [
        # one short question, 124M model: latency counts
        {"name": "prompt_short", "kind": "prompt", "f16": False, "seqs": 1, "heads": 12, "kv": 12, "low": 17, "high": 17, "past": 0},
        # one prompt of nearly the whole context, 124M model
        {"name": "prompt_one", "kind": "prompt", "f16": False, "seqs": 1, "heads": 12, "kv": 12, "low": 1001, "high": 1001, "past": 0},
        # sixteen prompts of different lengths at the 1.5B model's width
        {"name": "prompt_batch", "kind": "prompt", "f16": False, "seqs": 16, "heads": 25, "kv": 25, "low": 100, "high": 1023, "past": 0},
        # forty short turns of conversations of which 700 positions are there already, fp16 rows, four heads to a key head
        {"name": "prompt_turns_f16", "kind": "prompt", "f16": True, "seqs": 40, "heads": 16, "kv": 4, "low": 20, "high": 60, "past": 700},
        # one long document, fp16 rows, four heads to a key head
        {"name": "prompt_long_f16", "kind": "prompt", "f16": True, "seqs": 1, "heads": 16, "kv": 4, "low": 8001, "high": 8001, "past": 0},
        # one token of each of eight beams, 124M model
        {"name": "append_token", "kind": "append", "f16": False, "seqs": 8, "kv": 12, "start": 703, "low": 1, "high": 1, "max_seq": CTX},
        # sixteen packed prompts into the cache of the 1.5B model
        {"name": "append_prompts", "kind": "append", "f16": False, "seqs": 16, "kv": 25, "start": 0, "low": 100, "high": 1023, "max_seq": CTX},
        # a decode step's attention of eight beams that share a prompt and parts of what followed, 124M model
        {"name": "attend_beams", "kind": "attend", "seqs": 8, "heads": 12, "kv": 12, "low": 901, "high": 901, "max_seq": CTX, "beams": 8},
        # 48 sequences of different lengths at the 1.5B model's width
        {"name": "attend_batch", "kind": "attend", "seqs": 48, "heads": 25, "kv": 25, "low": 256, "high": CTX, "max_seq": CTX, "beams": 0},
        # one long sequence, four heads to a key head: the positions have to be split over the chip
        {"name": "attend_long", "kind": "attend", "seqs": 1, "heads": 16, "kv": 4, "low": 50001, "high": 50001, "max_seq": 65536, "beams": 0},
        # the smallest beam search
        {"name": "beam_four", "kind": "beam", "groups": 1, "beams": 4, "V": VOCAB, "T": 301, "max_seq": CTX},
        # sixteen texts with eight beams each, long tables
        {"name": "beam_many", "kind": "beam", "groups": 16, "beams": 8, "V": VOCAB, "T": 1001, "max_seq": CTX},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "prompt", "append", "attend", "attend", "beam"])
    heads = rng.choice([12, 16, 20, 25])
    kv = heads if rng.random() < 0.5 else heads // rng.choice([d for d in (2, 4, 5) if heads % d == 0])
    if kind == "prompt":
        f16 = rng.random() < 0.5
        high = _log(rng, 1, 6000 if f16 and rng.random() < 0.3 else CTX - 1)
        low = high if rng.random() < 0.3 else max(1, high // rng.choice([2, 4, 10]))
        past = rng.choice([0, 0, 0, rng.randint(1, 900), -rng.randint(1, 3)])
        most = 7000000 // (high * (high + 2 * max(past, 0)))  # (pairs of rows and keys: no more than the longest listed batch)
        return {"kind": kind, "f16": f16, "seqs": _log(rng, 1, max(1, min(16 if high > 100 else 40, most))), "heads": heads, "kv": kv,
                "low": low, "high": high, "past": past}
    if kind == "append":
        high = 1 if rng.random() < 0.4 else _log(rng, 2, 1000)
        return {"kind": kind, "f16": rng.random() < 0.5, "seqs": _log(rng, 1, 16), "kv": kv, "start": rng.randint(0, CTX - 1 - high),
                "low": max(1, high // 4), "high": high, "max_seq": CTX}
    if kind == "attend":
        if rng.random() < 0.3:
            T = _log(rng, 1500, 50000)
            return {"kind": kind, "seqs": max(1, min(rng.choice([1, 1, 2, 7]), 50000 * 4 // (T * kv))), "heads": heads,
                    "kv": kv if T * kv <= 50000 * 12 else 4 if heads % 4 == 0 else 5, "low": T, "high": T, "max_seq": T + rng.randint(0, 999), "beams": 0}
        beams = rng.choice([0, 0, 3, 4, 8])
        T = _log(rng, 4, CTX)
        return {"kind": kind, "seqs": beams * rng.randint(1, 4) or _log(rng, 1, 48), "heads": heads, "kv": kv, "low": T if beams else max(1, T // 4),
                "high": T, "max_seq": CTX, "beams": beams}
    return {"kind": kind, "groups": _log(rng, 1, 16), "beams": rng.randint(1, 8), "V": VOCAB if rng.random() < 0.5 else _log(rng, 1000, VOCAB),
            "T": rng.randint(1, CTX - 1), "max_seq": CTX}


def _lengths(c):
    """Lengths of a case's sequences between its bounds, long and short ones mixed."""
    n, low, high = c["seqs"], c["low"], c["high"]
    return [high if n == 1 else low + (high - low) * (i * 7 % n) // (n - 1) for i in range(n)]


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


# ------------------------------------------------------------------ 4-bit cache: layout

def _levels(dtype=torch.float32):
    half = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    return torch.tensor(half + [-v for v in half], device=DEV, dtype=dtype)


def _to4(x):
    """(codes [..., 64], bf16 scales [..., 2]) of fp32 rows x [..., 64]."""
    w = x.unflatten(-1, (2, 32))
    s = (w.abs().amax(-1) / torch.full((), 6.0, device=DEV)).bfloat16()
    q = w / s.float().clamp_min(1e-38).unsqueeze(-1)
    a = q.abs()
    # the eight magnitudes' borders; a border itself goes to the even code
    c = (a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    return torch.where((q < 0) & (c > 0), c + 8, c).flatten(-2), s


def _from4(codes, s, dtype=torch.float32):
    return (_levels(dtype)[codes.int()].unflatten(-1, (2, 32)) * s.to(dtype).unsqueeze(-1)).flatten(-2)


def _tiles(n):
    return -(-n // TILE)


def _cache_parts(cache, S, KV, max_seq):
    """Views of the cache's buffer [S, KV, tiles, 2304 bytes]: codes [..., K and V, 32, 32 bytes], scales [..., K and V, 32, 2]."""
    t = cache.view(S, KV, _tiles(max_seq), TILE_BYTES)
    n = 2 * TILE * DH // 2
    return t[..., :n].unflatten(-1, (2, TILE, DH // 2)), t[..., n:].view(torch.bfloat16).unflatten(-1, (2, TILE, 2))


def _values(state, dtype):
    """Keys and values that a cache stands for, [S, KV, 2, positions, 64], from the sequences that hold them."""
    c = state["c"]
    S, KV, n = c["seqs"], c["kv"], _tiles(c["high"])
    codes, scales = _cache_parts(state["cache"], S, KV, c["max_seq"])
    codes, scales = codes[:, :, :n].transpose(2, 3).flatten(3, 4), scales[:, :, :n].transpose(2, 3).flatten(3, 4)
    x = _from4(torch.stack([codes & 15, codes >> 4], -1).flatten(-2), scales, dtype)
    if c["beams"]:
        at = state["origin"][:, :n * TILE].long()  # whose slot a position is in
        if at.shape[1] < n * TILE:
            at = torch.nn.functional.pad(at, (0, n * TILE - at.shape[1]))
        x = torch.gather(x, 0, at[:, None, None, :, None].expand_as(x))
    return x


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(DEV).manual_seed(int(seed))


def prepare(case, seed):
    c, g = case, _gen(seed)

    def acts(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    def zeros(*shape, dtype=torch.float32):
        return torch.zeros(shape, device=DEV, dtype=dtype)

    def ints(values):
        return torch.tensor(values, device=DEV, dtype=torch.int32)

    s, k = {"c": c}, c["kind"]
    if k == "prompt":
        H, KV, lens = c["heads"], c["kv"], _lengths(c)
        keys = [max(0, n + c["past"]) for n in lens]
        t = torch.float16 if c["f16"] else torch.float32
        rows, key_rows = sum(lens) + SLACK, sum(keys) + SLACK
        qkv = acts(rows, (H + 2 * KV) * DH).to(t)  # what the product of the attention's input gives
        s["qkv"], s["q"] = qkv, qkv[:, :H * DH]
        if c["past"]:  # keys and values that were there before stand in front of the new ones
            s["kv"] = acts(key_rows, 2 * KV * DH).to(t)
            s["k"], s["v"] = s["kv"][:, :KV * DH], s["kv"][:, KV * DH:]
        else:
            s["k"], s["v"] = qkv[:, H * DH:(H + KV) * DH], qkv[:, (H + KV) * DH:]
        s["q_start"], s["k_start"] = ints(_starts(lens)), ints(_starts(keys))
        s["out"] = zeros(rows, H * DH, dtype=t)
    elif k == "append":
        KV, lens = c["kv"], _lengths(c)
        s["kv"] = acts(sum(lens) + SLACK, 2 * KV * DH).to(torch.float16 if c["f16"] else torch.float32)
        s["row_start"], s["pos"] = ints(_starts(lens)), ints([c["start"]] * c["seqs"])
        s["len"] = ints([c["start"] + n for n in lens])
        s["cache"] = zeros(c["seqs"] * KV * _tiles(c["max_seq"]) * TILE_BYTES, dtype=torch.uint8)
        s["k"], s["v"] = zeros(c["seqs"], c["high"], KV * DH), zeros(c["seqs"], c["high"], KV * DH)
        s["k_in"], s["v_in"] = s["kv"][:, :KV * DH], s["kv"][:, KV * DH:]
    elif k == "attend":
        S, H, KV, lens = c["seqs"], c["heads"], c["kv"], _lengths(c)
        s["cache"] = zeros(S * KV * _tiles(c["max_seq"]) * TILE_BYTES, dtype=torch.uint8)
        codes, scales = _cache_parts(s["cache"], S, KV, c["max_seq"])
        n = _tiles(c["high"])
        for i in range(S):
            q, sc = _to4(acts(KV, n, 2, TILE, DH))
            codes[i, :, :n], scales[i, :, :n] = q[..., 0::2] | (q[..., 1::2] << 4), sc
        s["q"], s["out"] = acts(S, (H + 2 * KV) * DH), zeros(S, H * DH)
        s["len"] = ints(lens)
        if c["beams"]:  # the prompt is the first beam's, what followed was continued from any beam
            first = torch.arange(S, device=DEV) // c["beams"] * c["beams"]
            at = first[:, None] + torch.randint(0, c["beams"], (S, c["max_seq"]), generator=g, device=DEV)
            at[:, :2 * c["high"] // 3] = first[:, None]
            s["origin"] = at.int()
        s["work"] = zeros(S * H * SPLITS * (2 + DH))
    else:
        G, B, V = c["groups"], c["beams"], c["V"]
        s["logits"] = 4 * acts(G * B, V)
        s["score"] = -20 + 2 * acts(G * B)
        s["done"] = (torch.rand(G * B, generator=g, device=DEV) < 0.1).int()
        s["ids"] = torch.randint(0, V, (G * B, c["max_seq"]), generator=g, device=DEV, dtype=torch.int32)
        group = torch.arange(G, device=DEV).repeat_interleave(B)[:, None] * B
        s["origin"] = (group + torch.randint(0, B, (G * B, c["max_seq"]), generator=g, device=DEV)).int()
        s["len"] = ints([c["T"]] * G)
        for n in ("new_score", "parent", "next", "new_done"):
            s[n] = zeros(G * B, dtype=torch.float32 if n == "new_score" else torch.int32)
        s["new_ids"], s["new_origin"] = zeros(G * B, c["max_seq"], dtype=torch.int32), zeros(G * B, c["max_seq"], dtype=torch.int32)
        s["work"] = zeros(_beam_bytes(c), dtype=torch.uint8) if own else None
    s["p"] = {n: t.data_ptr() for n, t in s.items() if isinstance(t, torch.Tensor)}
    return s


# ------------------------------------------------------------------ the framework's calls

_lib = []


def _g2():
    if not _lib:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gpt2-opencl-1.1_amd"))
        import g2hip

        g2hip.init(0)
        _lib.append(g2hip)
    return _lib[0]


def _beam_bytes(c):
    return _g2().beam_work_bytes(c["groups"], c["beams"], c["V"], c["beams"])


def _run_own(s):
    g2, c, p = _g2(), s["c"], s["p"]
    k = c["kind"]
    if k == "prompt":
        H, KV = c["heads"], c["kv"]
        g2.attn_prompt(p["q"], (H + 2 * KV) * DH, p["k"], p["v"], s["k"].stride(0), p["out"], H * DH, g2.F16 if c["f16"] else g2.F32,
                       p["q_start"], p["k_start"], c["seqs"], s["q"].shape[0], s["k"].shape[0], H, KV, SCALE)
        return s["out"]
    if k == "append":
        S, KV, n = c["seqs"], c["kv"], c["high"]
        g2.kv4_append(p["k_in"], p["v_in"], 2 * KV * DH, g2.F16 if c["f16"] else g2.F32, p["cache"], p["row_start"], p["pos"], 0, S,
                      s["kv"].shape[0], KV, c["max_seq"])
        g2.kv4_read(p["cache"], p["k"], p["v"], None, p["len"], c["start"] + n, c["start"], n, S, KV, c["max_seq"])
        return s["k"], s["v"]
    if k == "attend":
        H, KV = c["heads"], c["kv"]
        g2.attn_kv4(p["q"], (H + 2 * KV) * DH, p["cache"], p["out"], H * DH, p["origin"] if c["beams"] else None, p["len"], c["high"], c["seqs"],
                    H, KV, c["max_seq"], SCALE, p["work"])
        return s["out"]
    G, B, n = c["groups"], c["beams"], c["max_seq"]
    g2.beam_select(p["logits"], p["score"], p["done"], c["V"] - 1, p["new_score"], p["parent"], p["next"], p["new_done"], G, B, c["V"], B, p["work"])
    g2.beam_reorder(p["ids"], p["new_ids"], n, p["next"], p["origin"], p["new_origin"], n, p["parent"], p["len"], c["T"], G, B)
    return s["new_score"], s["parent"], s["next"], s["new_done"], s["new_ids"], s["new_origin"]


# ------------------------------------------------------------------ plain form

def _seq_heads(x, H):
    """Rows [n, H * 64] as [H, n, 64]."""
    return x.reshape(x.shape[0], H, DH).transpose(0, 1)


def _run_plain(s):
    c = s["c"]
    k = c["kind"]
    if k == "prompt":
        out = torch.zeros(s["out"].shape, device=DEV)
        lens = _lengths(c)
        qs, ks = _starts(lens), _starts([max(0, n + c["past"]) for n in lens])
        H, KV = c["heads"], c["kv"]
        for i in range(c["seqs"]):
            a, b = slice(qs[i], qs[i + 1]), slice(ks[i], ks[i + 1])
            n, m = qs[i + 1] - qs[i], ks[i + 1] - ks[i]
            if not m:
                continue
            seen = torch.arange(m, device=DEV) <= torch.arange(n, device=DEV)[:, None] + (m - n)
            q = _seq_heads(s["q"][a].float(), H)
            key, val = _seq_heads(s["k"][b].float(), KV), _seq_heads(s["v"][b].float(), KV)
            for h in range(KV):  # (a key head's scores at a time: long prompts' would not fit otherwise)
                r = slice(h * (H // KV), (h + 1) * (H // KV))
                w = (q[r] @ key[h].t()) * SCALE
                w = w.masked_fill(~seen, -INF)
                w = torch.exp(w - w.amax(2, keepdim=True).clamp_min(-1e30))
                o = (w / w.sum(2, keepdim=True).clamp_min(1e-30)) @ val[h]
                out[a].view(n, H, DH)[:, r] = o.transpose(0, 1)
        return out.to(s["out"].dtype)
    if k == "append":
        lens = _lengths(c)
        at, out = _starts(lens), []
        for x in (s["k_in"], s["v_in"]):
            codes, sc = _to4(x.float().reshape(x.shape[0], c["kv"], DH))
            y, r = _from4(codes, sc).reshape(x.shape[0], -1), torch.zeros_like(s["k"])
            for i, n in enumerate(lens):
                r[i, :n] = y[at[i]:at[i + 1]]
            out.append(r)
        return tuple(out)
    if k == "attend":
        S, H, KV = c["seqs"], c["heads"], c["kv"]
        kv = _values(s, torch.float32)
        q = s["q"][:, :H * DH].reshape(S, KV, H // KV, DH)
        w = (q @ kv[:, :, 0].transpose(2, 3).contiguous()) * SCALE
        w = w.masked_fill((torch.arange(kv.shape[3], device=DEV) >= s["len"][:, None])[:, None, None], -INF)
        w = torch.exp(w - w.amax(3, keepdim=True))
        return ((w / w.sum(3, keepdim=True)) @ kv[:, :, 1].contiguous()).reshape(S, H * DH)
    G, B, V = c["groups"], c["beams"], c["V"]
    l = s["logits"].double()  # (candidates' order: 32 bits would make ties)
    top = l.amax(1, keepdim=True)
    total = s["score"].double()[:, None] + (l - top - torch.log(torch.exp(l - top).sum(1, keepdim=True)))
    # an ended beam goes on as it is
    over = s["done"].bool()[:, None]
    total = torch.where(over, torch.full_like(total, -INF), total)
    total[:, V - 1] = torch.where(over[:, 0], s["score"].double(), total[:, V - 1])
    total = total.view(G, B * V)
    got, score = [], []
    for _ in range(B):
        best = total.amax(1, keepdim=True)
        i = torch.where(total == best, torch.arange(B * V, device=DEV), B * V).amin(1, keepdim=True)
        total.scatter_(1, i, -INF)
        got.append(i)
        score.append(best)
    return _moved(s, torch.cat(score, 1), torch.cat(got, 1))


def _moved(s, score, flat):
    """Scores and flat candidates [groups, beams] as the step's outputs."""
    c = s["c"]
    G, B, V, T = c["groups"], c["beams"], c["V"], c["T"]
    parent, token = flat // V, flat % V
    row = (parent + B * torch.arange(G, device=DEV)[:, None]).reshape(-1)
    done = s["done"][row].bool() | (token.reshape(-1) == V - 1)
    ids, origin = torch.zeros_like(s["ids"]), torch.zeros_like(s["origin"])
    ids[:, :T], origin[:, :T] = s["ids"][row, :T], s["origin"][row, :T]
    ids[:, T], origin[:, T] = token.reshape(-1).int(), torch.arange(G * B, device=DEV, dtype=torch.int32)
    score = score.reshape(-1)
    return score if score.dtype == torch.float64 and s.get("wide") else score.float(), parent.reshape(-1).int(), token.reshape(-1).int(), \
        done.int(), ids, origin


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s, c = prepare(case, seed), case
    k = c["kind"]
    if k == "prompt":
        out = torch.zeros(s["out"].shape, device=DEV, dtype=torch.float64)
        at = kt = 0
        for n in _lengths(c):
            m = max(0, n + c["past"])
            for h in range(c["heads"]):
                f = h // (c["heads"] // c["kv"]) * DH
                key, val = s["k"][kt:kt + m, f:f + DH].double(), s["v"][kt:kt + m, f:f + DH].double()
                first = max(0, n - m)  # rows before it see no key
                for r in range(first, n, 2048):
                    e = min(n, r + 2048)
                    x = s["q"][at + r:at + e, h * DH:(h + 1) * DH].double() @ key.t() / 8
                    behind = torch.ones(e - r, m, device=DEV, dtype=torch.bool).triu(m - n + r + 1)
                    out[at + r:at + e, h * DH:(h + 1) * DH] = torch.softmax(x.masked_fill_(behind, -INF), 1) @ val
            at, kt = at + n, kt + m
        return out
    if k == "append":
        out = [torch.zeros(s["k"].shape, device=DEV, dtype=torch.float64) for _ in range(2)]
        up = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=DEV, dtype=torch.float64)
        for x, r in zip((s["k_in"], s["v_in"]), out):
            # by the definition: the scale is a/6 rounded to fp32 and to bf16, the nearest of the 16 values to x/scale (fp32)
            w = x.double().reshape(x.shape[0], -1, 32)
            sc = (w.abs().amax(2, keepdim=True) / 6).float().bfloat16().double()
            q = torch.where(sc > 0, w / sc, torch.zeros_like(w)).float().double()
            i = torch.searchsorted(up, q.abs().clamp_max(6)).clamp(1, 7)  # between up[i - 1] and up[i]
            far, near = up[i] - q.abs().clamp_max(6), q.abs().clamp_max(6) - up[i - 1]
            i = torch.where((near < far) | ((near == far) & (i % 2 == 1)), i - 1, i)
            y, at = (up[i] * q.sign() * sc).reshape(x.shape[0], -1), 0
            for j, n in enumerate(_lengths(c)):
                r[j, :n] = y[at:at + n]
                at += n
        return tuple(out)
    if k == "attend":
        kv, out = _values(s, torch.float64), torch.zeros(s["out"].shape, device=DEV, dtype=torch.float64)
        for i, n in enumerate(_lengths(c)):
            for h in range(c["heads"]):
                x = kv[i, h // (c["heads"] // c["kv"]), :, :n]
                w = torch.softmax((x[0] * s["q"][i, h * DH:(h + 1) * DH].double()).sum(1) / 8, 0)
                out[i, h * DH:(h + 1) * DH] = (w[:, None] * x[1]).sum(0)
        return out
    G, B, V = c["groups"], c["beams"], c["V"]
    t = torch.log_softmax(s["logits"].double(), 1) + s["score"].double()[:, None]
    t[s["done"] == 1] = -INF
    t[s["done"] == 1, V - 1] = s["score"].double()[s["done"] == 1]
    score, flat = torch.sort(t.view(G, B * V), dim=1, descending=True, stable=True)
    s["wide"] = True
    return _moved(s, score[:, :B], flat[:, :B])


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    c, k = case, case["kind"]
    if k == "prompt":
        lens = _lengths(c)
        keys = [max(0, n + c["past"]) for n in lens]
        pairs = sum(sum(max(0, i + 1 + m - n) for i in range(n)) for n, m in zip(lens, keys))
        size = 2 if c["f16"] else 4
        return {"bytes": size * DH * (2 * c["heads"] * sum(lens) + 2 * c["kv"] * sum(keys)), "flops": 4 * DH * c["heads"] * pairs}
    if k == "append":
        n = 2 * c["kv"] * sum(_lengths(c))  # heads' rows of 64
        return {"bytes": n * ((2 if c["f16"] else 4) * DH + 2 * 36 + 4 * DH), "flops": 2 * n * DH}
    if k == "attend":
        n = sum(_lengths(c))
        held = n
        if c["beams"]:  # a group's first two thirds are shared, of the rest each beam may have its own
            T = c["high"]
            held = c["seqs"] // c["beams"] * (2 * T // 3) + c["seqs"] * (T - 2 * T // 3)
        return {"bytes": 72 * c["kv"] * held + 8 * DH * c["heads"] * c["seqs"] + (4 * n if c["beams"] else 0), "flops": 4 * DH * c["heads"] * n}
    R = c["groups"] * c["beams"]
    return {"bytes": 4 * R * c["V"] + 16 * R * c["T"] + 32 * R, "flops": 4 * R * c["V"]}
