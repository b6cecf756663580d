"""Operators of the 8-bit key/value cache: quantising as it is written, reading it back, and the attention that reads it.

A page holds 16 tokens; what a page keeps of one kv head is one record of bytes: codes of K (16 rows of head_dim), codes of V, 16 exponents
of K, 16 of V. A value is its code (fp8 e4m3, or a whole number of 8 bits) times 2^exponent; a token's row of a kv head has one exponent, the smallest
that keeps the row within the codes' range, stored with 127 added. Rows lie in pieces of 16 bytes; a piece's place is its number with some bits
turned over by the key it belongs to (`_places`).

`run` computes in 32 bits with elementary torch operations, or, where `own` is true, calls `infinilm_b200.ops`.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
PAGE = 16
TOP = {"fp8_e4m3": (0.875, 9), "int8": (0.9921875, 7)}        # the largest code, 448 and 127, as fraction and power of two
LEAST, MOST = -100, 100                           # exponents of a row


# ---- the cases ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a decode step of one request: rotate, quantise and write one token - the smallest call, all latency (8B sizes)
        _case("store_step_b1", "store", "fp8_e4m3", "bfloat16", 32, 2, 128, 1, 700, 700, 1, 1),
        # a decode step of 64 requests of the 0.5B sizes
        _case("store_step_b64", "store", "int8", "bfloat16", 16, 2, 64, 64, 20, 600, 1, 1),
        # prompts of a full step (token budget 8,192), some of them later portions of their request
        _case("store_prompts", "store", "fp8_e4m3", "bfloat16", 32, 8, 128, 6, 0, 2048, 555, 2048),
        # one short request read back
        _case("read_one", "read", "int8", "bfloat16", 16, 2, 64, 1, 333, 333, 0, 0),
        # a batch of long contexts read back
        _case("read_many", "read", "fp8_e4m3", "bfloat16", 32, 8, 128, 16, 1000, 8192, 0, 0),
        # one request of a small model behind a question: bound by launches
        _case("decode_b1_short", "decode", "fp8_e4m3", "bfloat16", 16, 2, 64, 1, 18, 18, 1, 1),
        # the headline benchmark's decode step: eight requests of 2,048 tokens, 32 heads on 2
        _case("decode_b8", "decode", "fp8_e4m3", "bfloat16", 32, 2, 128, 8, 2047, 2047, 1, 1),
        # one request with a very long context: the split over its length
        _case("decode_b1_long", "decode", "int8", "bfloat16", 32, 2, 128, 1, 131071, 131071, 1, 1),
        # a serving batch of unequal contexts: bound by memory
        _case("decode_b64", "decode", "fp8_e4m3", "bfloat16", 32, 8, 128, 64, 500, 8191, 1, 1),
        # one prompt of a small model
        _case("prompt_one", "prompt", "int8", "bfloat16", 16, 2, 64, 1, 0, 0, 600, 600),
        # later portions of several requests, each behind what it has cached
        _case("prompts_behind", "prompt", "fp8_e4m3", "bfloat16", 32, 2, 128, 5, 0, 4096, 37, 1024),
        # one prompt as long as a step's budget
        _case("prompt_8k", "prompt", "fp8_e4m3", "bfloat16", 32, 8, 128, 1, 0, 0, 8192, 8192),
    ]


def _case(name, op, kind, act, nh, nkv, hd, entries, cached_least, cached_most, new_least, new_most, window=0):
    return {"name": name, "op": op, "kind": kind, "act": act, "heads": nh, "kv_heads": nkv, "head_dim": hd, "entries": entries,
            "cached_least": cached_least, "cached_most": cached_most, "new_least": new_least, "new_most": new_most, "window": window}


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["store", "read", "decode", "prompt"])
    kind = rng.choice(["fp8_e4m3", "int8"])
    nh, nkv, hd = rng.choice([(16, 2, 64), (12, 12, 64), (32, 2, 128), (16, 4, 128), (32, 8, 128), (64, 8, 128), (8, 8, 128), (20, 4, 64), (8, 2, 256)])
    act, window = "bfloat16", 0
    if op == "store":
        entries, most = rng.choice([(1, 8192), (_log(rng, 1, 64), 1), (_log(rng, 2, 8), 1024)])
        act = rng.choice(["bfloat16", "bfloat16", "float32"])
        new = _log(rng, 1, most)
        cached = _log(rng, 1, 20000) if entries == 1 else _log(rng, 1, 1500)
        c = (entries, cached // 2, cached, max(1, new // 3), new)
    elif op == "read":
        entries = _log(rng, 1, 16)
        act = rng.choice(["bfloat16", "float32"])
        n = _log(rng, 1, 8192 if act == "bfloat16" else 4000)
        c = (entries, max(1, n // 4), n, 0, 0)
    elif op == "decode":
        entries = _log(rng, 1, 64)
        n = _log(rng, 1, min(131071, 400000 // entries))
        window = rng.choice([0, 0, 0, _log(rng, 16, 4096)])
        c = (entries, n // 5, n, 1, 1)
    else:
        entries = _log(rng, 1, 6)
        new, cached = _log(rng, 2, 4096 // entries), _log(rng, 1, 6000 // entries)
        window = rng.choice([0, 0, 0, _log(rng, 16, 2048)])
        c = (entries, 0, cached, max(1, new // 4), new)
    case = _case("", op, kind, act, nh, nkv, hd, *c, window=window)
    del case["name"]
    return case


def _lengths(case):
    """Tokens in the cache before the call, and new ones, of every entry: the first has the most of both."""
    r = random.Random(case["entries"] * 1000003 + case["cached_most"] * 17 + case["new_most"])
    n = case["entries"]
    cached = [case["cached_most"]] + [r.randint(case["cached_least"], case["cached_most"]) for _ in range(n - 1)]
    new = [case["new_most"]] + [r.randint(case["new_least"], case["new_most"]) for _ in range(n - 1)]
    return cached, new


def _first_seen(pos, window):
    return max(0, pos - window + 1) if window > 0 else 0


def _sees(start, new, window):
    """Keys seen by the tokens start .. start + new - 1, added up."""
    if window <= 0 or start + new <= window:
        return new * start + new * (new + 1) // 2
    return sum(min(p + 1, window) for p in range(start, start + new))


def work(case):
    cached, new = _lengths(case)
    nh, nkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    act = 4 if case["act"] == "float32" else 2
    record, T, w = nkv * (2 * hd + 2), sum(new), case["window"]
    if case["op"] == "store":                     # written, and the tokens' pages read back as bfloat16
        back = sum(((s + n - 1) // PAGE - s // PAGE + 1) * PAGE for s, n in zip(cached, new))
        return {"bytes": T * ((2 * nh + 2 * nkv) * hd * act + record) + back * (record + 2 * nkv * hd * 2), "flops": T * (nh + nkv) * hd * 3}
    if case["op"] == "read":
        return {"bytes": sum(cached) * (record + 2 * nkv * hd * act), "flops": 0}
    keys = sum(s + n - _first_seen(s, w) for s, n in zip(cached, new))
    pairs = sum(_sees(s, n, w) for s, n in zip(cached, new))
    return {"bytes": keys * record + 2 * T * nh * hd * act, "flops": 4 * pairs * nh * hd}


# ---- what a user's program has in hand -------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    cached, new = _lengths(case)
    nh, nkv, hd, kind, E = case["heads"], case["kv_heads"], case["head_dim"], case["kind"], case["entries"]
    act = torch.float32 if case["act"] == "float32" else torch.bfloat16
    kvlen = [s + n for s, n in zip(cached, new)]
    width = max((n + PAGE - 1) // PAGE for n in kvlen)
    need = [(n + PAGE - 1) // PAGE for n in kvlen]
    n_pages = sum(need) + 1
    # pages that were handed out and given back for a while: in no order; every slot holds something, behind a request's end too
    order = torch.randperm(n_pages, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((E, width), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for e in range(E):
        table[e, :need[e]] = order[at:at + need[e]]
        at += need[e]
    # keys have a few large columns that all tokens share, values a size of their own for every token
    cols = torch.exp(0.6 * torch.randn((nkv, 1, hd), generator=g, device=DEVICE))
    cache = torch.empty((n_pages, nkv, 32 * hd + 32), dtype=torch.uint8, device=DEVICE)
    for a in range(0, n_pages, 2048):
        b = min(n_pages, a + 2048)
        k = torch.randn((b - a, nkv, PAGE, hd), generator=g, device=DEVICE) * cols
        v = torch.randn((b - a, nkv, PAGE, hd), generator=g, device=DEVICE)
        v *= torch.exp(0.5 * torch.randn((b - a, nkv, PAGE, 1), generator=g, device=DEVICE))
        cache[a:b] = _records(k.to(torch.bfloat16).float(), v.to(torch.bfloat16).float(), kind)
    s = {"case": dict(case), "kind": kind, "cache": cache, "table": table, "cached": cached, "new": new, "kvlen_host": kvlen, "width": width,
         "kvlen": torch.tensor(kvlen, dtype=torch.int32, device=DEVICE), "act": act, "dims": (nh, nkv, hd), "window": case["window"],
         "scale": 1.0 / math.sqrt(hd)}
    T = sum(new)
    qstart = [0]
    for n in new:
        qstart.append(qstart[-1] + n)
    s["qstart"] = torch.tensor(qstart, dtype=torch.int32, device=DEVICE)
    if T:
        s["entry"] = torch.repeat_interleave(torch.arange(E, device=DEVICE), torch.tensor(new, device=DEVICE)).to(torch.int32)
        within = torch.arange(T, device=DEVICE) - s["qstart"][:-1][s["entry"].long()]
        s["pos"] = (within + torch.tensor(cached, device=DEVICE)[s["entry"].long()]).to(torch.int32)
    if case["op"] == "store":
        s["inv_freq"] = (1.0 / 10000.0 ** (torch.arange(0, hd, 2, dtype=torch.float64) / hd)).float().to(DEVICE)
        s["qkv"] = torch.randn((T, (nh + 2 * nkv) * hd), generator=g, device=DEVICE).to(act)
        s["q_out"] = torch.empty((T, nh * hd), dtype=act, device=DEVICE)
        s["pages"] = torch.zeros((E * width, 2, nkv, PAGE, hd), dtype=torch.bfloat16, device=DEVICE)
    elif case["op"] == "read":
        s["pages"] = torch.zeros((E * width, 2, nkv, PAGE, hd), dtype=act, device=DEVICE)
    else:
        s["q"] = (1.5 * torch.randn((T, nh * hd), generator=g, device=DEVICE)).to(act)
        s["out"] = torch.empty((T, nh * hd), dtype=act, device=DEVICE)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------
def _places(hd, device):
    """Where the 16-byte pieces of K's rows and of V's lie in their plane: two tables [16 keys, head_dim / 16]."""
    key = torch.arange(PAGE, device=device)[:, None]
    number = key * (hd // 16) + torch.arange(hd // 16, device=device)[None, :]
    turned = hd in (64, 128, 256)
    return (number ^ ((key & 1) << 2) if turned and hd > 64 else number), (number ^ (((key >> 1) & 3) << 1) if turned else number)


def _quantise(x, kind):
    """Codes as bytes and exponents as bytes of rows x [..., head_dim] in 32 bits."""
    top, power = TOP[kind]
    most = x.abs().amax(-1, keepdim=True)
    part, exp = torch.frexp(most)
    e = exp - power + (part > top)
    e = torch.where(most == 0, torch.zeros_like(e), e.clamp(min=LEAST))
    bad = ~torch.isfinite(most) | (e > MOST)
    e = torch.where(bad, torch.zeros_like(e), e)
    y = torch.where(bad, torch.zeros_like(x), torch.ldexp(x, -e))
    code = y.to(torch.float8_e4m3fn).view(torch.uint8) if kind == "fp8_e4m3" else torch.round(y).to(torch.int8).view(torch.uint8)
    return code, torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)[..., 0]


def _records(k, v, kind):
    """Whole pages k, v [pages, kv_heads, 16, head_dim] as records."""
    P, nkv, _, hd = k.shape
    out = torch.empty((P, nkv, 32 * hd + 32), dtype=torch.uint8, device=k.device)
    for i, (x, place) in enumerate(zip((k, v), _places(hd, k.device))):
        code, e = _quantise(x, kind)
        plane = torch.empty((P, nkv, hd, 16), dtype=torch.uint8, device=k.device)
        plane[:, :, place.reshape(-1)] = code.reshape(P, nkv, hd, 16)
        out[:, :, i * 16 * hd:(i + 1) * 16 * hd] = plane.reshape(P, nkv, 16 * hd)
        out[:, :, 32 * hd + 16 * i:32 * hd + 16 * i + 16] = e
    return out


def _power(e):
    """2^(byte - 127) in 32 bits; 255: not a number."""
    return torch.where(e == 255, torch.full_like(e, math.nan, dtype=torch.float32), (e.to(torch.int32) << 23).view(torch.float32))


def _values(records, hd, kind):
    """K and V [..., 16, head_dim] in 32 bits of records [..., bytes]."""
    lead, got = records.shape[:-1], []
    for i, place in enumerate(_places(hd, records.device)):
        code = records[..., i * 16 * hd:(i + 1) * 16 * hd].reshape(*lead, hd, 16)[..., place.reshape(-1), :].reshape(*lead, PAGE, hd)
        code = code.view(torch.float8_e4m3fn if kind == "fp8_e4m3" else torch.int8).float()
        got.append(code * _power(records[..., 32 * hd + 16 * i:32 * hd + 16 * i + 16])[..., None])
    return got


def _read(s, first, dtype):
    """The entries' pages from token first[e] on as values [entries * width, 2, kv_heads, 16, head_dim]; zero in front of that page and behind the end."""
    _, nkv, hd = s["dims"]
    k, v = _values(s["cache"][s["table"].long().clamp(min=0)], hd, s["kind"])      # [entries, width, kv_heads, 16, head_dim]
    key = torch.arange(s["width"] * PAGE, device=k.device).view(1, s["width"], PAGE)
    there = (key < s["kvlen"][:, None, None]) & (key >= (first // PAGE * PAGE)[:, None, None])
    both = torch.stack([k, v], dim=2)
    return torch.where(there[:, :, None, None, :, None], both, torch.zeros_like(both)).to(dtype).reshape(-1, 2, nkv, PAGE, hd)


def _store_plain(s):
    nh, nkv, hd = s["dims"]
    x = s["qkv"].float().view(-1, nh + 2 * nkv, hd)
    angle = s["pos"].double()[:, None] * s["inv_freq"].double()[None, :]          # far positions: in 64 bits
    c, sn = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    x1, x2 = x[:, :nh + nkv, :hd // 2], x[:, :nh + nkv, hd // 2:]
    turned = torch.cat([x1 * c - x2 * sn, x2 * c + x1 * sn], dim=-1)
    q = turned[:, :nh].to(s["act"]).reshape(-1, nh * hd)
    entry, pos = s["entry"].long(), s["pos"].long()
    page, slot = s["table"].long()[entry, pos // PAGE][:, None], (pos % PAGE)[:, None]
    head = torch.arange(nkv, device=q.device)[None, :]
    cache, places = s["cache"], _places(hd, q.device)
    for i, rows in enumerate((turned[:, nh:], x[:, nh + nkv:])):                  # K, then V
        code, e = _quantise(rows, s["kind"])
        plane = cache[:, :, i * 16 * hd:(i + 1) * 16 * hd].view(-1, nkv, hd, 16)
        plane[page[..., None], head[..., None], places[i][slot[:, 0]][:, None, :]] = code.reshape(-1, nkv, hd // 16, 16)
        cache[page, head, 32 * hd + 16 * i + slot] = e
    return {"q": q, "pages": _read(s, torch.tensor(s["cached"], device=q.device), torch.bfloat16)}


def _attend_plain(s):
    nh, nkv, hd = s["dims"]
    G, E, W = nh // nkv, len(s["new"]), s["width"]
    k, v = (x.transpose(1, 2).reshape(E, nkv, W * PAGE, hd) for x in _values(s["cache"][s["table"].long().clamp(min=0)], hd, s["kind"]))
    most = max(s["new"])
    within = torch.arange(most, device=k.device)
    there = within[None, :] < torch.tensor(s["new"], device=k.device)[:, None]                # [entries, most]
    row = (s["qstart"][:-1].long()[:, None] + within[None, :]).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[row].view(E, most, nkv, G, hd).permute(0, 2, 1, 3, 4).reshape(E, nkv, most * G, hd)
    score = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).view(E, nkv, most, G, W * PAGE)
    pos = torch.tensor(s["cached"], device=k.device)[:, None] + within[None, :]
    key = torch.arange(W * PAGE, device=k.device)[None, None, :]
    hidden = key > pos[:, :, None]
    if s["window"] > 0:
        hidden |= key <= (pos - s["window"])[:, :, None]
    score.masked_fill_(hidden[:, None, :, None, :], -math.inf)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.view(E, nkv, most * G, W * PAGE), v).view(E, nkv, most, G, hd) / total
    return out.permute(0, 2, 1, 3, 4).reshape(E, most, nh * hd)[there].to(s["act"])


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        return _run_own(s, op)
    if op == "store":
        return _store_plain(s)
    if op == "read":
        return _read(s, torch.zeros_like(s["kvlen"]), s["act"])
    return _attend_plain(s)


# ---- the framework's operators -------------------------------------------------------------------------------------------------------
def _run_own(s, op):
    from infinilm_b200 import ops
    nh, nkv, hd = s["dims"]
    if op == "store":
        ops.rope_store_quant(s["qkv"], s["q_out"], s["pos"], s["entry"], s["table"], s["cache"], s["kind"], nh, nkv, hd, hd, s["inv_freq"], 1.0)
        ops.kv_unpack(s["cache"], s["kind"], s["table"], s["kvlen"], s["pages"], entry_qstart=s["qstart"], window=1)
        return {"q": s["q_out"], "pages": s["pages"]}
    if op == "read":
        ops.kv_unpack(s["cache"], s["kind"], s["table"], s["kvlen"], s["pages"])
        return s["pages"]
    if "ws" not in s:                             # buffers that the program keeps from step to step
        from infinilm_b200.engine.step import Workspace
        s["ws"] = Workspace(DEVICE, 8192)
    if op == "decode":
        ops.attention_decode_quant(s["q"], s["out"], s["cache"], s["kind"], s["table"], s["kvlen"], len(s["new"]), nh, nkv, hd, s["scale"],
                                   s["window"], max(s["kvlen_host"]), s["ws"])
    else:
        per = ops.prefill_quant_tokens(nh, nkv, hd)
        ops.attention_prefill_quant(s["q"], s["out"], s["cache"], s["kind"], s["table"], s["qstart"], s["kvlen"], 0, len(s["new"]),
                                    sum((n + per - 1) // per for n in s["new"]), nh, nkv, hd, s["scale"], s["window"], s["ws"])
    return s["out"]


# ---- in 64 bits, by the definition -------------------------------------------------------------------------------------------------------
def _exact_rows(s, e):
    """K and V of entry e in 64 bits, [kv_heads, kvlen, head_dim], byte by byte of its records."""
    _, nkv, hd = s["dims"]
    n = s["kvlen_host"][e]
    t = torch.arange(n, device=DEVICE)
    page, key = s["table"][e].long()[t // PAGE], t % PAGE
    col = torch.arange(hd, device=DEVICE)
    piece = key[:, None] * (hd // 16) + col[None, :] // 16
    got = []
    for i in (0, 1):
        turn = torch.zeros_like(key)
        if i == 0 and hd in (128, 256):
            turn = (key % 2) * 4
        elif i == 1 and hd in (64, 128, 256):
            turn = (key // 2 % 4) * 2
        byte = torch.bitwise_xor(piece, turn[:, None]) * 16 + col[None, :] % 16 + i * 16 * hd
        codes = torch.gather(s["cache"][page], 2, byte[:, None, :].expand(n, nkv, hd)).to(torch.int64)
        if s["kind"] == "int8":
            code = torch.where(codes > 127, codes - 256, codes).double()
        else:
            power, part = codes // 8 % 16, codes % 8
            code = torch.where(power == 0, part.double() * 2.0 ** -9, (8 + part).double() * 2.0 ** (power.double() - 10))
            code = torch.where(codes > 127, -code, code)
        e8 = torch.gather(s["cache"][page], 2, (32 * hd + 16 * i + key)[:, None, None].expand(n, nkv, 1)).double()
        got.append((code * 2.0 ** (e8 - 127)).transpose(0, 1))
    return got


def exact(case, seed):
    s = prepare(case, seed)
    nh, nkv, hd = s["dims"]
    if case["op"] == "store":                     # the queries; what the cache holds is a choice among codes, which has no such value
        x = s["qkv"].double().view(-1, nh + 2 * nkv, hd)[:, :nh]
        z = torch.polar(torch.ones((), dtype=torch.float64, device=DEVICE), s["pos"].double()[:, None] * s["inv_freq"].double())[:, None]
        z = torch.complex(x[..., :hd // 2].contiguous(), x[..., hd // 2:].contiguous()) * z
        return {"q": torch.cat([z.real, z.imag], dim=-1).reshape(-1, nh * hd), "pages": None}
    if case["op"] == "read":
        pages = torch.zeros(s["pages"].shape, dtype=torch.float64, device=DEVICE)
        for e in range(case["entries"]):
            n = s["kvlen_host"][e]
            t = torch.arange(n, device=DEVICE)
            for i, x in enumerate(_exact_rows(s, e)):
                pages[e * s["width"] + t // PAGE, i, :, t % PAGE] = x.transpose(0, 1)
        return pages
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for e in range(case["entries"]):
        k, v = _exact_rows(s, e)
        a, n, start = int(s["qstart"][e]), s["new"][e], s["cached"][e]
        pos, key = torch.arange(start, start + n, device=DEVICE)[:, None], torch.arange(k.shape[1], device=DEVICE)[None, :]
        seen = (key <= pos) if s["window"] <= 0 else (key <= pos) & (key > pos - s["window"])
        for h in range(nh):
            score = s["q"][a:a + n, h * hd:(h + 1) * hd].double() @ k[h // (nh // nkv)].T / math.sqrt(hd)
            out[a:a + n, h * hd:(h + 1) * hd] = torch.softmax(score.masked_fill(~seen, -math.inf), dim=-1) @ v[h // (nh // nkv)]
    return out
