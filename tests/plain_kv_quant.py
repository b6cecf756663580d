"""The 8-bit key/value cache in 64 bits, by its definition: codes and exponents of rows, records of pages, values of records, and attention over them."""
import math

import numpy as np
import torch

PAGE = 16
TOP = {"fp8_e4m3": 448.0, "int8": 127.0}


def e4m3_values():
    """The 256 codes' values (NaN for 127 and 255)."""
    v = np.empty(256)
    for c in range(256):
        power, part = c >> 3 & 15, c & 7
        x = part * 2.0 ** -9 if power == 0 else (8 + part) * 2.0 ** (power - 10)
        v[c] = math.nan if c & 127 == 127 else -x if c & 128 else x
    return v


def exponents(x, kind):
    """The byte of every row of x [..., head_dim] (float64)."""
    most = x.abs().amax(-1)
    top = TOP[kind]
    e = torch.ceil(torch.log2(torch.where((most > 0) & torch.isfinite(most), most, torch.ones_like(most)) / top))
    # (the logarithm is rounded: the smallest e that holds, looked for around it)
    e = torch.where(most <= top * torch.pow(2.0, e - 1), e - 1, e)
    e = torch.where(most > top * torch.pow(2.0, e), e + 1, e)
    e = torch.where(most == 0, torch.zeros_like(e), e.clamp(min=-100))
    bad = ~torch.isfinite(most) | (e > 100)
    return torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.int64)


def step(x, byte, kind):
    """The distance of neighbouring codes' values around x of a row with that byte."""
    unit = torch.pow(2.0, byte.double() - 127)[..., None]
    if kind == "int8":
        return unit.expand(x.shape)
    mag = (x.abs() / unit).clamp(min=2.0 ** -6)
    return unit * torch.pow(2.0, torch.floor(torch.log2(mag)) - 3)


def encode(x, kind):
    """Values (float64) and bytes of the rows x [..., head_dim] as the cache holds them; rounding half to even."""
    byte = exponents(x, kind)
    bad = (byte == 255)[..., None]
    unit = torch.pow(2.0, byte.double() - 127)[..., None]
    y = torch.where(bad, torch.zeros_like(x), x / unit)
    if kind == "int8":
        r = torch.round(y)
    else:
        grid = torch.pow(2.0, torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        r = torch.round(y / grid) * grid
    return torch.where(bad, torch.full_like(x, math.nan), r * unit), byte


def place(hd, v, key, chunk):
    number = key * (hd // 16) + chunk
    if v and hd in (64, 128, 256):
        return number ^ (key // 2 % 4 * 2)
    if not v and hd in (128, 256):
        return number ^ (key % 2 * 4)
    return number


def record_index(hd):
    """Byte of (K or V, key, column) in a record, [2, 16, head_dim]."""
    at = torch.empty((2, PAGE, hd), dtype=torch.int64)
    for v in (0, 1):
        for key in range(PAGE):
            for chunk in range(hd // 16):
                a = v * PAGE * hd + 16 * place(hd, v, key, chunk)
                at[v, key, 16 * chunk:16 * chunk + 16] = torch.arange(a, a + 16)
    return at


def decode_records(records, hd, kind):
    """Values [..., 2, 16, head_dim] in 64 bits of records uint8 [..., 32 head_dim + 32] (on the CPU)."""
    codes = records[..., record_index(hd).reshape(-1)].reshape(*records.shape[:-1], 2, PAGE, hd).to(torch.int64)
    table = torch.from_numpy(e4m3_values()) if kind == "fp8_e4m3" else torch.tensor([float(c - 256 if c > 127 else c) for c in range(256)], dtype=torch.float64)
    byte = records[..., 32 * hd:].reshape(*records.shape[:-1], 2, PAGE, 1).double()
    unit = torch.where(byte == 255, torch.full_like(byte, math.nan), torch.pow(2.0, byte - 127))
    return table[codes] * unit


def make_records(kv, kind):
    """Records uint8 [pages, kv_heads, bytes] of values kv [pages, kv_heads, 2, 16, head_dim] (any float, rounded as the cache rounds)."""
    x = kv.double()
    hd = x.shape[-1]
    val, byte = encode(x, kind)
    unit = torch.pow(2.0, byte.double() - 127)[..., None]
    y = torch.nan_to_num(val / unit, nan=0.0)
    if kind == "int8":
        codes = y.to(torch.int64) & 255
    else:
        order = torch.from_numpy(np.where(np.isnan(e4m3_values()), 1e9, e4m3_values()))
        pos = order[:127]                         # ascending magnitudes
        codes = torch.searchsorted(pos, y.abs().contiguous()) + 128 * (y < 0)
    out = torch.empty((*x.shape[:2], 32 * hd + 32), dtype=torch.uint8)
    out[..., record_index(hd).reshape(-1)] = codes.reshape(*x.shape[:2], -1).to(torch.uint8)
    out[..., 32 * hd:] = byte.reshape(*x.shape[:2], 32).to(torch.uint8)
    return out


def mask_lo(pos, window):
    if window > 0:
        return max(0, pos - window + 1)
    return pos - pos % -window if window < 0 else 0


def attend(q, kv, table_row, pos, scale, window):
    """One token's heads q [heads, head_dim] at `pos` over values kv [pages, kv_heads, 2, 16, head_dim]: output and sum of weight times |value| (both [heads,
    head_dim]); a page below 0 is masked; no key: zeros."""
    nh, nkv = q.shape[0], kv.shape[1]
    keys = [t for t in range(mask_lo(pos, window), pos + 1) if table_row[t // PAGE] >= 0]
    if not keys:
        z = torch.zeros(q.shape, dtype=torch.float64)
        return z, z
    t = torch.tensor(keys)
    rows = kv[torch.as_tensor(table_row)[t // PAGE].long(), :, :, t % PAGE]       # [keys, kv_heads, 2, head_dim]
    out, mag = [], []
    for h in range(nh):
        k, v = rows[:, h // (nh // nkv), 0].double(), rows[:, h // (nh // nkv), 1].double()
        p = torch.softmax(k @ q[h].double() * scale, 0)
        out.append(p @ v)
        mag.append(p @ v.abs())
    return torch.stack(out), torch.stack(mag)
