"""The 8-bit key/value cache on the device against its definition in 64 bits: writing, reading back, attention of single tokens and of prompt
portions, and all of them in a row."""
import math

import pytest
import torch

import plain_kv_quant as P

pytestmark = pytest.mark.gpu
KINDS = ["fp8_e4m3", "int8"]


def _ops():
    from infinilm_b200 import ops
    return ops


def _ws(dev, tokens=256):
    from infinilm_b200.engine.step import Workspace
    return Workspace(dev, tokens)


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _tables(kvlens, spare, seed, width=None):
    """Block table rows over shuffled pages, and the number of pages."""
    need = [(n + 15) // 16 for n in kvlens]
    g = torch.Generator().manual_seed(seed)
    ids = torch.randperm(sum(need) + spare, generator=g).tolist()
    width = width or max(1, max(need))
    rows, at = [], 0
    for n in need:
        rows.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    return rows, sum(need) + spare


def _cache(n_pages, nkv, hd, kind, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    kv = torch.randn((n_pages, nkv, 2, 16, hd), generator=g) * torch.exp(spread * torch.randn((n_pages, nkv, 2, 16, 1), generator=g))
    rec = P.make_records(kv, kind)
    return rec, P.decode_records(rec, hd, kind)


# ---- writing ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh,nkv,hd,rot", [(4, 2, 64, 64), (3, 1, 128, 128), (2, 2, 256, 256), (5, 5, 16, 16), (4, 2, 48, 24), (4, 2, 80, 32), (2, 1, 112, 0),
                                           (4, 1, 192, 96), (2, 1, 128, 6), (36, 4, 64, 64)])
@pytest.mark.parametrize("T", [1, 7, 130])
def test_store_rounds_each_row_to_its_codes(cuda_device, kind, dtype, nh, nkv, hd, rot, T):
    ops, dev = _ops(), cuda_device
    g = torch.Generator().manual_seed(T * 31 + hd)
    qkv = (torch.randn((T, (nh + 2 * nkv) * hd), generator=g) * torch.exp(2 * torch.randn((T, 1), generator=g))).to(dtype)
    start, half = 5, rot // 2
    rows, n_pages = _tables([start + T], 3, 1)
    inv = (1.0 / 10000.0 ** (torch.arange(half).double() / max(half, 1))).float()
    cache = torch.full((n_pages, nkv, ops.kv_quant_record(hd)), 0xA5, dtype=torch.uint8, device=dev)
    q = torch.zeros((T, nh * hd), dtype=dtype, device=dev)
    src = qkv.to(dev)
    pos = torch.arange(start, start + T)
    ops.rope_store_quant(src, q, _i32(pos.tolist(), dev), _i32([0] * T, dev), _i32(rows, dev), cache, kind, nh, nkv, hd, rot, inv.to(dev), 1.25)
    assert torch.equal(src.cpu(), qkv)            # the rows are left as they were
    x = qkv.double().view(T, nh + 2 * nkv, hd)
    ang = pos.double()[:, None] * inv.double()
    c, s = 1.25 * torch.cos(ang)[:, None], 1.25 * torch.sin(ang)[:, None]
    turned = x.clone()
    qk = slice(0, nh + nkv)
    turned[:, qk, :half], turned[:, qk, half:rot] = x[:, qk, :half] * c - x[:, qk, half:rot] * s, x[:, qk, half:rot] * c + x[:, qk, :half] * s
    # sine and cosine within 3 units of 2^-24 and an angle reduced to 2^-22, two products and a sum rounded: 2^-20 of the pair's size
    size = turned.abs()
    size[:, qk, :half] = size[:, qk, half:rot] = x[:, qk, :half].abs() + x[:, qk, half:rot].abs()
    slack = size * 1.25 * 2.0 ** -20 * (rot > 0)
    eps = torch.finfo(dtype).eps / 2
    got_q = q.cpu().double().view(T, nh, hd)
    assert ((got_q - turned[:, :nh]).abs() <= turned[:, :nh].abs() * eps * (1 + 2.0 ** -10) + slack[:, :nh] * (1 + eps)).all()
    got = P.decode_records(cache.cpu(), hd, kind)
    byte = cache.cpu()[..., 32 * hd:].reshape(n_pages, nkv, 2, 16)
    page, key = torch.tensor(rows[0])[pos // 16], pos % 16
    val, b = got[page, :, :, key], byte[page, :, :, key].long()                   # [T, nkv, 2, hd], [T, nkv, 2]
    want = torch.stack([turned[:, nh:nh + nkv], x[:, nh + nkv:]], 2)
    room = torch.stack([slack[:, nh:nh + nkv], torch.zeros_like(x[:, nh + nkv:])], 2)
    most = want.abs().amax(-1)
    lo, hi = P.exponents((want.abs() - room).clamp(min=0), kind), P.exponents(want.abs() + room, kind)
    assert ((b >= torch.minimum(lo, hi)) & (b <= hi)).all() and (most > 0).all()
    assert ((val - want).abs() <= P.step(want, b, kind) / 2 * (1 + 2.0 ** -18) + room).all()
    exact, be = P.encode(want[:, :, 1], kind)     # V is not turned: bit for bit
    assert torch.equal(val[:, :, 1], exact) and torch.equal(b[:, :, 1], be)
    if rot == 0:
        assert torch.equal(val[:, :, 0], P.encode(want[:, :, 0], kind)[0])
    touched = torch.zeros(n_pages, 16, dtype=torch.bool)
    touched[page, key] = True
    at = P.record_index(hd)
    for p in range(n_pages):                      # every other slot is left as it was
        rest = cache[p].cpu()
        codes, exps = rest[:, at.reshape(-1)].reshape(nkv, 2, 16, hd), rest[:, 32 * hd:].reshape(nkv, 2, 16)
        assert (codes[:, :, ~touched[p]] == 0xA5).all() and (exps[:, :, ~touched[p]] == 0xA5).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [1, 200])
def test_store_in_place_strided_and_without_a_cache(cuda_device, kind, T):
    """q may be written over its own columns; rows may have a stride; a page that is not there is not stored to; without a cache only q is made."""
    ops, dev = _ops(), cuda_device
    nh, nkv, hd = 4, 2, 64
    g = torch.Generator().manual_seed(T)
    w = (nh + 2 * nkv) * hd
    qkv = torch.randn((T, w), generator=g).to(torch.bfloat16).to(dev)
    inv = torch.rand(hd // 2, generator=g).to(dev)
    rows, n_pages = _tables([T], 1, 2)
    pos, ent = _i32(list(range(T)), dev), _i32([0] * T, dev)
    cache, q = torch.zeros((n_pages, nkv, ops.kv_quant_record(hd)), dtype=torch.uint8, device=dev), torch.empty((T, nh * hd), dtype=torch.bfloat16, device=dev)
    ops.rope_store_quant(qkv, q, pos, ent, _i32(rows, dev), cache, kind, nh, nkv, hd, hd, inv, 1.0)
    wide = torch.zeros((T, w + 24), dtype=torch.bfloat16, device=dev)
    wide[:, :w] = qkv
    other = torch.zeros_like(cache)
    ops.rope_store_quant(wide[:, :w], wide[:, :nh * hd], pos, ent, _i32(rows, dev), other, kind, nh, nkv, hd, hd, inv, 1.0)
    assert torch.equal(wide[:, :nh * hd], q) and torch.equal(other, cache) and torch.equal(wide[:, nh * hd:w], qkv[:, nh * hd:]) and not wide[:, w:].any()
    odd = torch.zeros((T * w + 3,), dtype=torch.bfloat16, device=dev)[3:].view(T, w)        # not on a 16-byte boundary
    odd.copy_(qkv)
    other.zero_()
    ops.rope_store_quant(odd, odd[:, :nh * hd], pos, ent, _i32(rows, dev), other, kind, nh, nkv, hd, hd, inv, 1.0)
    assert torch.equal(odd[:, :nh * hd], q) and torch.equal(other, cache)
    other.fill_(7)
    q2 = torch.empty_like(q)
    ops.rope_store_quant(qkv, q2, pos, ent, _i32([[-1] * len(rows[0])], dev), other, kind, nh, nkv, hd, hd, inv, 1.0)
    ops.rope_store_quant(qkv, q2, pos, ent, _i32(rows, dev), None, kind, nh, nkv, hd, hd, inv, 1.0)
    assert torch.equal(q2, q) and (other == 7).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [9, 108])
def test_store_of_rows_at_the_ends_of_the_range(cuda_device, kind, T):
    """Zeros, the largest code and the next value above it, ties, rows that are not finite, too large or too small."""
    ops, dev = _ops(), cuda_device
    hd, top = 64, P.TOP[kind]
    x = torch.zeros((9, hd), dtype=torch.float32)
    x[1, 3], x[1, 4] = top * 2.0 ** 5, -1.0
    x[2, 3], x[2, 4:12] = top * 2.0 ** 5 * (1 + 2.0 ** -23), torch.tensor([1.0, -2.5, 3.5, 0.03125, 17.0, -18.0, 19.0, 33.0]) * 64
    x[3] = torch.arange(hd) / 2.0                 # halves: ties of whole numbers
    x[3, 0] = 127.0
    x[4, 5], x[4, 6] = math.inf, 1.0
    x[5, 5], x[5, 6] = math.nan, 1.0
    x[6, 0] = 3e38
    x[7, 0], x[7, 1] = 1e-33, 1e-38
    x[8, 0] = top * 2.0 ** 100
    x = x.repeat(T // 9, 1)
    qkv = torch.cat([torch.zeros((T, hd)), x, x.flip(1)], 1).to(dev)
    rows, n_pages = _tables([T], 1, 3)
    cache = torch.zeros((n_pages, 1, ops.kv_quant_record(hd)), dtype=torch.uint8, device=dev)
    q = torch.empty((T, hd), device=dev)
    ops.rope_store_quant(qkv, q, _i32(list(range(T)), dev), _i32([0] * T, dev), _i32(rows, dev), cache, kind, 1, 1, hd, 0, None, 1.0)
    t = torch.arange(T)
    got = P.decode_records(cache.cpu(), hd, kind)[torch.tensor(rows[0])[t // 16], 0, :, t % 16]
    for i, y in enumerate((x, x.flip(1))):
        want, byte = P.encode(y.double(), kind)
        assert torch.equal(got[:, i].nan_to_num(nan=123.0), want.nan_to_num(nan=123.0))
    assert byte[:9].tolist()[4:7] == [255, 255, 255] and byte[0] == 127 and byte[8] == 227


def test_far_positions_turn_by_the_exact_angle(cuda_device):
    ops, dev = _ops(), cuda_device
    hd, pos = 128, [0, 1, 4095, 131071, 1000003, 2 ** 30]
    T = len(pos)
    inv = (1.0 / 10000.0 ** (torch.arange(64).double() / 64)).float()
    x = torch.randn((T, 3 * hd), generator=torch.Generator().manual_seed(0))
    q = torch.empty((T, hd), device=dev)
    ops.rope_store_quant(x.to(dev), q, _i32(pos, dev), _i32([0] * T, dev), _i32([[0]], dev), None, "int8", 1, 1, hd, hd, inv.to(dev), 1.0)
    ang = torch.tensor(pos).double()[:, None] * inv.double()
    a, b = x[:, :64].double(), x[:, 64:128].double()
    want = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], 1)
    size = torch.cat([a.abs() + b.abs()] * 2, 1)
    assert ((q.cpu().double() - want).abs() <= size * 2.0 ** -20).all()


# ---- reading back -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nkv,hd", [(2, 64), (1, 128), (3, 256), (2, 16), (1, 80), (2, 192)])
def test_unpack_gives_the_values_exactly(cuda_device, kind, dtype, nkv, hd):
    ops, dev = _ops(), cuda_device
    kvlens = [0, 1, 15, 16, 17, 50, 33]
    rows, n_pages = _tables(kvlens, 2, 4)
    rows[5][1] = -1                               # a page that is not there
    rec, val = _cache(n_pages, nkv, hd, kind, 5, spread=3.0)
    rec[rows[6][0], 0, 32 * hd + 3], rec[rows[6][1], nkv - 1, 32 * hd + 16 + 9] = 255, 255       # a row of K, one of V that are NaN
    val = P.decode_records(rec, hd, kind)
    W = len(rows[0])
    cache, tab, kvl = rec.to(dev), _i32(rows, dev), _i32(kvlens, dev)
    pages = torch.full((len(kvlens) * W, 2, nkv, 16, hd), 77.0, dtype=dtype, device=dev)
    table = torch.full_like(tab, -5)
    ops.kv_unpack(cache, kind, tab, kvl, pages, table)
    assert table.cpu().tolist() == [[e * W + p for p in range(W)] for e in range(len(kvlens))]
    got = pages.cpu().double().view(len(kvlens), W, 2, nkv, 16, hd)

    def check(got, first, special):
        for e, n in enumerate(kvlens):
            for p in range(W):
                if p * 16 >= n or p < first[e]:
                    assert (got[e, p] == 77.0).all()
                    continue
                want = torch.zeros((2, nkv, 16, hd), dtype=torch.float64)
                if rows[e][p] >= 0:
                    want = val[rows[e][p]].transpose(0, 1).clone()
                    special(e, p, want)
                want[:, :, min(16, n - p * 16):] = 0.0
                assert torch.equal(got[e, p].nan_to_num(nan=1e9), want.nan_to_num(nan=1e9))
    check(got, [0] * 7, lambda e, p, w: None)

    def moved(e, p, w):                           # V's NaN is told by its key
        if e == 6 and p == 1:
            w[0, nkv - 1, 9], w[1, nkv - 1, 9] = math.nan, 0.0
    pages.fill_(77.0)
    ops.kv_unpack(cache, kind, tab, kvl, pages, None, nan_in_keys=True)
    check(pages.cpu().double().view(len(kvlens), W, 2, nkv, 16, hd), [0] * 7, moved)
    # only what new tokens see: entries with 2 new tokens, a window of 5; entries from the third on
    qs = _i32([0, 0, 0, 2, 4, 6, 8, 10], dev)
    pages.fill_(77.0)
    table.fill_(-5)
    ops.kv_unpack(cache, kind, tab, kvl, pages, table, entry_qstart=qs, window=5, first_entry=2)
    got = pages.cpu().double().view(len(kvlens), W, 2, nkv, 16, hd)
    assert (got[5:] == 77.0).all() and (table.cpu()[:2] == -5).all() and table.cpu()[2].tolist() == list(range(W))
    first = [max(0, n - 2 - 4) // 16 for n in kvlens]
    check(torch.cat([torch.full_like(got[:2], 77.0), got[:5]]), [9, 9] + first[2:], lambda e, p, w: None)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [5, 300])
def test_unpack_packed(cuda_device, kind, n):
    """The pages that are seen one behind the other, for more requests than a block has threads too; what has no room is left out and reported."""
    ops, dev = _ops(), cuda_device
    nkv, hd = 1, 64
    g = torch.Generator().manual_seed(n)
    kvlens = [0, 40, 16, 1, 33] + torch.randint(0, 50, (n - 5,), generator=g).tolist()
    new = [min(k, 2) for k in kvlens]
    rows, n_pages = _tables(kvlens, 1, 21, width=5)
    rec, val = _cache(n_pages, nkv, hd, kind, 22)
    qs = [0]
    for x in new:
        qs.append(qs[-1] + x)
    window = 10
    first = [max(0, k - x - window + 1) // 16 for k, x in zip(kvlens, new)]
    seen = [max(0, (k + 15) // 16 - f) for k, f in zip(kvlens, first)]
    total = sum(seen[1:])
    tab, kvl = _i32(rows, dev), _i32(kvlens, dev)
    ops.check_status(dev)
    for room in (total, total + 3, total - 1):
        pages, table = torch.full((room + 1, 2, nkv, 16, hd), 77.0, device=dev), torch.full_like(tab, -5)
        ops.kv_unpack(rec.to(dev), kind, tab, kvl, pages[:room], table, entry_qstart=_i32(qs, dev), window=window, first_entry=1, packed=True)
        at = 0
        got, where = pages.cpu().double(), table.cpu()
        for e in range(1, n):
            for p in range(5):
                if not first[e] <= p < first[e] + seen[e]:
                    assert where[e, p] == 0
                    continue
                if at >= room:
                    assert where[e, p] == 0
                else:
                    assert where[e, p] == at
                    k = min(16, kvlens[e] - 16 * p)
                    assert torch.equal(got[at][:, :, :k], val[rows[e][p]].transpose(0, 1)[:, :, :k]) and not got[at][:, :, k:].any()
                at += 1
        assert (got[min(at, room):] == 77.0).all() and (where[0] == -5).all()
        if room < total:
            with pytest.raises(ops.KernelError, match="kv_quant"):
                ops.check_status(dev)
        else:
            ops.check_status(dev)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,dtype", [(16, torch.bfloat16), (64, torch.float32), (128, torch.bfloat16)])
@pytest.mark.parametrize("window", [None, 20, -32])
def test_unpack_with_wide_tables(cuda_device, kind, hd, dtype, window):
    """Many requests with tables far wider than they need (the pages are then dealt out to blocks): what narrow tables give, packed and by place."""
    ops, dev = _ops(), cuda_device
    n, nkv, narrow, wide = 300, 2, 6, 40
    g = torch.Generator().manual_seed(hd)
    kvlens = [0 if i % 5 == 2 else int(torch.randint(0, 90, (1,), generator=g)) for i in range(n)]
    kvlens[0], kvlens[299] = 96, 95
    new = [min(k, 1 + i % 3) for i, k in enumerate(kvlens)]
    qs = [0]
    for x in new:
        qs.append(qs[-1] + x)
    rows, n_pages = _tables(kvlens, 0, 21, width=narrow)
    cache = _cache(n_pages, nkv, hd, kind, 22)[0].to(dev)
    rest = dict(entry_kvlen=_i32(kvlens, dev), entry_qstart=_i32(qs, dev), window=window)
    got = []
    for width in (narrow, wide):
        tab = _i32([r + [-1] * (width - narrow) for r in rows], dev)
        for first in (0, 7):
            pages, table = torch.full((n_pages, 2, nkv, 16, hd), 77.0, dtype=dtype, device=dev), torch.full_like(tab, -5)
            ops.kv_unpack(cache, kind, tab, pages=pages, table=table, first_entry=first, packed=True, **rest)
            placed, by_place = torch.full((n * width, 2, nkv, 16, hd), 77.0, dtype=dtype, device=dev), torch.full_like(tab, -5)
            ops.kv_unpack(cache, kind, tab, pages=placed, table=by_place, first_entry=first, **rest)
            assert not table[first:, narrow:].any() and (table[:first] == -5).all() and (by_place[:first] == -5).all()
            assert torch.equal(by_place[first:].cpu(), torch.arange((n - first) * width, dtype=torch.int32).view(n - first, width))
            spare = placed[(n - first) * width:]
            assert (spare == 77.0).all() and (placed[:(n - first) * width].view(n - first, width, -1)[:, narrow:] == 77.0).all()
            got.append((pages, table[first:, :narrow], placed[:(n - first) * width].view(n - first, width, -1)[:, :narrow]))
    for a, b in ((0, 2), (1, 3)):
        assert all(torch.equal(x, y) for x, y in zip(got[a], got[b]))
    ops.check_status(dev)
    few = torch.full((5, 2, nkv, 16, hd), 77.0, dtype=dtype, device=dev)
    table = torch.full_like(tab, -5)
    ops.kv_unpack(cache, kind, tab, pages=few[:4], table=table, packed=True, **rest)
    assert torch.equal(few[:4], got[0][0][:4]) and (few[4] == 77.0).all() and int(table.max()) == 3
    with pytest.raises(ops.KernelError, match="kv_quant"):
        ops.check_status(dev)


# ---- single tokens -----------------------------------------------------------------------------------------------------------
def _decode_check(out, q, val, rows, kvlens, nh, hd, scale, window):
    for e, n in enumerate(kvlens):
        want, mag = P.attend(q[e].view(nh, hd), val, rows[e], n - 1, scale, window) if n > 0 else (torch.zeros((nh, hd)).double(),) * 2
        # the output's rounding; weights as halves: 2^-11 each (below 2^-14 of the largest: 2^-25); exponentials, exponents and sums in 32 bits: 2^-15 together
        room = want.abs() * 2.0 ** -8 * (1 + 2.0 ** -8) + mag * (2.0 ** -11 + 2.0 ** -15) + 2.0 ** -25 * mag.amax(-1, keepdim=True) * max(n, 1)
        got = out[e].double().view(nh, hd)
        assert ((got - want).abs() <= room).all(), (e, n, ((got - want).abs() / room.clamp(min=1e-300)).max())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nh,nkv,hd", [(16, 2, 64), (4, 4, 64), (32, 2, 128), (6, 2, 128), (20, 1, 128), (8, 2, 256), (40, 1, 64)])
@pytest.mark.parametrize("blocks", [0, 1, 2, 7, 300, -2, -4, -8])
@pytest.mark.parametrize("window", [None, 20, -24])
def test_decode_over_codes(cuda_device, monkeypatch, kind, nh, nkv, hd, blocks, window):
    ops, dev = _ops(), cuda_device
    kvlens = [300, 1, 0, 16, 17, 129, 15, 47]
    rows, n_pages = _tables(kvlens, 3, 6)
    rec, val = _cache(n_pages, nkv, hd, kind, 7)
    for e, n in enumerate(kvlens):                # behind a request's end anything may lie: codes and exponents that are NaN
        if n % 16:
            k = torch.arange(n % 16, 16)
            rec[rows[e][n // 16]][:, P.record_index(hd)[:, k].reshape(-1)] = 0x7F
            rec[rows[e][n // 16]][:, torch.cat([32 * hd + k, 32 * hd + 16 + k])] = 255
    g = torch.Generator().manual_seed(8)
    q = (2 * torch.randn((len(kvlens), nh * hd), generator=g)).to(torch.bfloat16)
    q[:, :hd] *= 2.0 ** 20                        # a head far outside what a half holds
    q[:, hd:2 * hd] *= 2.0 ** -30
    monkeypatch.setattr(ops, "_quant_blocks", lambda *a: blocks)
    out = torch.full((len(kvlens), nh * hd), 3.0, dtype=torch.bfloat16, device=dev)
    scale = 0.7 / math.sqrt(hd)
    for early in (False, True):
        out.fill_(3.0)
        ops.attention_decode_quant(q.to(dev), out, rec.to(dev), kind, _i32(rows, dev), _i32(kvlens, dev), len(kvlens), nh, nkv, hd, scale, window, 300, _ws(dev),
                                   cached_before=early)
        _decode_check(out.cpu(), q, val, rows, kvlens, nh, hd, scale, window or 0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("blocks", [0, 5, 23, -2, -8])
def test_decode_pages_that_are_not_there_and_rows_that_are_not_finite(cuda_device, monkeypatch, kind, hd, blocks):
    """A missing page's keys are masked, a request without any page gets zeros; a NaN row reaches the heads and requests that see it, no others; exponents far apart."""
    ops, dev = _ops(), cuda_device
    nh, nkv, kvlens = 4, 2, [70, 40, 33, 64, 90]
    rows, n_pages = _tables(kvlens, 1, 9)
    rows[0][1] = rows[0][4] = -1
    rows[1] = [-1] * len(rows[1])
    g = torch.Generator().manual_seed(10)
    kv = torch.randn((n_pages, nkv, 2, 16, hd), generator=g)
    last = rows[4]
    kv[torch.tensor(last[:6]), :, 1] *= torch.exp2(torch.randint(-40, 40, (6, nkv, 16, 1), generator=g).float())      # values' exponents far apart
    kv[last[3], 1, 1, 5] = 0.0
    kv[last[2], 0, 0, 3] = 0.0
    rec = P.make_records(kv, kind)
    val = P.decode_records(rec, hd, kind)
    rec[rows[2][0], 1, 32 * hd + 16 + 3] = 255    # V of kv head 1, key 3 of request 2: NaN
    rec[rows[3][1], 0, 32 * hd + 7] = 255         # K of kv head 0, key 23 of request 3: NaN
    q = torch.randn((5, nh * hd), generator=g).to(torch.bfloat16)
    monkeypatch.setattr(ops, "_quant_blocks", lambda *a: blocks)
    out = torch.full((5, nh * hd), 3.0, dtype=torch.bfloat16, device=dev)

    def go(window):
        ops.attention_decode_quant(q.to(dev), out, rec.to(dev), kind, _i32(rows, dev), _i32(kvlens, dev), 5, nh, nkv, hd, 1.0 / math.sqrt(hd), window, 90, _ws(dev))
        return out.cpu()
    got = go(None)
    assert not got[1].any()
    assert torch.isnan(got[2, 2 * hd:]).all() and torch.isnan(got[3, :2 * hd]).all()
    got[2, 2 * hd:], got[3, :2 * hd] = 0, 0
    for e in (0, 1, 4):
        _decode_check(got[e:e + 1], q[e:e + 1], val, rows[e:e + 1], kvlens[e:e + 1], nh, hd, 1.0 / math.sqrt(hd), 0)
    _decode_check(got[2:3, :2 * hd], q[2:3, :2 * hd], val[:, :1], rows[2:3], kvlens[2:3], 2, hd, 1.0 / math.sqrt(hd), 0)
    got = go(25)                                  # the NaN rows lie in front of the window
    assert not torch.isnan(got).any()
    _decode_check(got[2:4], q[2:4], val, rows[2:4], kvlens[2:4], nh, hd, 1.0 / math.sqrt(hd), 25)


def test_decode_takes_rows_with_a_stride_and_is_repeatable(cuda_device):
    ops, dev = _ops(), cuda_device
    nh, nkv, hd, kvlens = 32, 2, 128, [2000, 700, 1999]
    rows, n_pages = _tables(kvlens, 0, 11)
    rec = torch.randint(0, 120, (n_pages, nkv, ops.kv_quant_record(hd)), dtype=torch.uint8, generator=torch.Generator().manual_seed(1)).to(dev)
    rec[..., 32 * hd:] = 120
    wide = torch.randn((3, (nh + 2 * nkv) * hd), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(dev)
    tab, kvl, ws, outs = _i32(rows, dev), _i32(kvlens, dev), _ws(dev), []
    for q in (wide, wide[:, :nh * hd], wide[:, :nh * hd].contiguous(), wide):
        out = torch.empty((3, nh * hd), dtype=torch.bfloat16, device=dev)
        ops.attention_decode_quant(q, out, rec, "int8", tab, kvl, 3, nh, nkv, hd, 0.05, None, 2000, ws)
        outs.append(out)
    assert all(torch.equal(o, outs[0]) for o in outs[1:])
    ops.check_status(dev)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("blocks", [16, 17, 100, 600, -8])
def test_decode_of_long_contexts_in_many_parts(cuda_device, monkeypatch, kind, hd, blocks):
    """Parts by the hundred of one unit, beside requests of a page; the same bits twice."""
    ops, dev = _ops(), cuda_device
    nh, nkv, kvlens = 2, 1, [3, 5000, 16, 2001]
    rows, n_pages = _tables(kvlens, 2, 18)
    rec, val = _cache(n_pages, nkv, hd, kind, 19)
    q = torch.randn((4, nh * hd), generator=torch.Generator().manual_seed(20)).to(torch.bfloat16)
    monkeypatch.setattr(ops, "_quant_blocks", lambda *a: blocks)
    ws, outs = _ws(dev), []
    for _ in range(2):
        out = torch.full((4, nh * hd), 3.0, dtype=torch.bfloat16, device=dev)
        ops.attention_decode_quant(q.to(dev), out, rec.to(dev), kind, _i32(rows, dev), _i32(kvlens, dev), 4, nh, nkv, hd, 0.1, None, 5000, ws)
        outs.append(out.cpu())
    assert torch.equal(outs[0], outs[1])
    _decode_check(outs[0], q, val, rows, kvlens, nh, hd, 0.1, 0)


def test_offsets_past_32_bits(cuda_device):
    """A cache of more than 4 GB: a request whose pages lie at its far end."""
    ops, dev = _ops(), cuda_device
    nh, nkv, hd, n = 8, 8, 128, 40
    rec_bytes = nkv * ops.kv_quant_record(hd)
    n_pages = (1 << 32) // rec_bytes + 100
    cache = torch.empty((n_pages, nkv, ops.kv_quant_record(hd)), dtype=torch.uint8, device=dev)
    rows = [[n_pages - 1, n_pages - 7, n_pages - 3]]
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn((n, (nh + 2 * nkv) * hd), generator=g).to(torch.bfloat16).to(dev)
    q = torch.empty((n, nh * hd), dtype=torch.bfloat16, device=dev)
    tab, kvl = _i32(rows, dev), _i32([n], dev)
    ops.rope_store_quant(qkv, q, _i32(list(range(n)), dev), _i32([0] * n, dev), tab, cache, "int8", nh, nkv, hd, 0, None, 1.0)
    pages = torch.empty((3, 2, nkv, 16, hd), dtype=torch.float32, device=dev)
    ops.kv_unpack(cache, "int8", tab, kvl, pages)
    v = pages[:, 1].transpose(1, 2).reshape(48, nkv, hd)[:n].cpu().double()
    assert torch.equal(v, P.encode(qkv[:, (nh + nkv) * hd:].cpu().double().view(n, nkv, hd), "int8")[0])
    out = torch.empty((1, nh * hd), dtype=torch.bfloat16, device=dev)
    ops.attention_decode_quant(q[-1:], out, cache, "int8", tab, kvl, 1, nh, nkv, hd, 0.1, None, n, _ws(dev))
    val = pages.cpu().double().transpose(1, 2)
    _decode_check(out.cpu(), q[-1:].cpu(), val, [[0, 1, 2]], [n], nh, hd, 0.1, 0)


# ---- prompt portions -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nh,nkv,hd", [(16, 2, 64), (4, 4, 128), (32, 2, 128), (4, 1, 256), (6, 2, 64)])
@pytest.mark.parametrize("window", [None, 40, -32])
@pytest.mark.parametrize("pair_from", [0, 1 << 30])
def test_prompt_portions_over_codes(cuda_device, monkeypatch, kind, nh, nkv, hd, window, pair_from):
    """With two row tiles a block and with one."""
    ops, dev = _ops(), cuda_device
    monkeypatch.setattr(ops, "PAIR_FROM", pair_from)
    cached, new = [9, 0, 100, 0, 31], [1, 37, 20, 1, 80]     # the first entry is a single token that another kernel takes
    kvlens = [a + b for a, b in zip(cached, new)]
    rows, n_pages = _tables(kvlens, 2, 12)
    rec, val = _cache(n_pages, nkv, hd, kind, 13, spread=0.5)
    bad = (rows[4][5], min(14, 90 - 80))          # a NaN row of V that the later tokens of entry 4 see, the earlier do not
    rec[bad[0], 0, 32 * hd + 16 + bad[1]] = 255
    rec[rows[2][7]][:, P.record_index(hd)[:, 9:].reshape(-1)] = 0x7F            # behind the end of entry 2
    T = sum(new)
    q = torch.randn((T, nh * hd), generator=torch.Generator().manual_seed(14)).to(torch.bfloat16)
    qs = [0]
    for n in new:
        qs.append(qs[-1] + n)
    per = ops.prefill_quant_tokens(nh, nkv, hd)
    out = torch.full((T, nh * hd), 3.0, dtype=torch.bfloat16, device=dev)
    scale = 1.0 / math.sqrt(hd)
    ops.attention_prefill_quant(q.to(dev), out, rec.to(dev), kind, _i32(rows, dev), _i32(qs, dev), _i32(kvlens, dev), 1, 5, sum((n + per - 1) // per for n in new[1:]),
                                nh, nkv, hd, scale, window, _ws(dev))
    got = out.cpu().double()
    assert (got[0] == 3.0).all()
    for e in range(1, 5):
        for i in range(0, new[e], 1 if new[e] < 30 else 7):
            pos, t = cached[e] + i, qs[e] + i
            want, mag = P.attend(q[t].view(nh, hd), val, rows[e], pos, scale, window or 0)
            row = got[t].view(nh, hd)
            if e == 4 and P.mask_lo(pos, window or 0) <= 90 <= pos:
                assert torch.isnan(row[:nh // nkv]).all()
                row, want, mag = row[nh // nkv:], want[nh // nkv:], mag[nh // nkv:]
            # the output's rounding, the weights' to bfloat16 (both 2^-8), the rest in 32 bits
            room = want.abs() * 2.0 ** -8 * (1 + 2.0 ** -8) + mag * (2.0 ** -8 + 2.0 ** -14)
            assert ((row - want).abs() <= room).all(), (e, i, ((row - want).abs() / room.clamp(min=1e-300)).max())
    ops.check_status(dev)


@pytest.mark.parametrize("pair_from", [0, 1 << 30])
@pytest.mark.parametrize("window", [None, 40])
def test_prompts_that_share_pages_and_prompts_that_do_not(cuda_device, monkeypatch, pair_from, window):
    """More pages seen than the cache has, as requests share them; and the room that requests with pages of their own need at most, which gives the same bits."""
    ops, dev = _ops(), cuda_device
    monkeypatch.setattr(ops, "PAIR_FROM", pair_from)
    nh, nkv, hd, E, n, kvlen = 4, 2, 64, 9, 5, 100
    rows, n_pages = _tables([kvlen], 0, 12)
    rec, _ = _cache(n_pages, nkv, hd, "int8", 13, spread=0.5)
    q = torch.randn((n, nh * hd), generator=torch.Generator().manual_seed(14)).to(torch.bfloat16).to(dev)
    per = ops.prefill_quant_tokens(nh, nkv, hd)

    def run(entries, **kw):
        out = torch.full((entries * n, nh * hd), 3.0, dtype=torch.bfloat16, device=dev)
        ops.attention_prefill_quant(q.repeat(entries, 1), out, rec.to(dev), "int8", _i32(rows * entries, dev), _i32([i * n for i in range(entries + 1)], dev), _i32([kvlen] * entries, dev),
                                    0, entries, entries * ((n + per - 1) // per), nh, nkv, hd, 0.125, window, _ws(dev), **kw)
        return out
    one, many = run(1), run(E)
    assert torch.equal(many.view(E, n, nh * hd), one.expand(E, n, nh * hd))
    cache = rec.to(dev)
    assert torch.equal(run(1, room=ops.unpacked_room(cache, 1, len(rows[0]))), one)
    ops.check_status(dev)
    run(2, room=(3 if window else 8))
    with pytest.raises(ops.KernelError, match="kv_quant"):
        ops.check_status(dev)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nh,nkv,hd", [(16, 2, 64), (8, 1, 128), (3, 1, 128), (2, 1, 256)])
@pytest.mark.parametrize("window", [None, 300])
@pytest.mark.parametrize("pair_from", [0, 1 << 30])
def test_long_portions_with_many_key_tiles(cuda_device, monkeypatch, kind, nh, nkv, hd, window, pair_from):
    """Chains of key tiles, rows of a block's two halves with chains of unequal length, large scores (the running maximum is raised tile after tile), a NaN that late tokens see."""
    ops, dev = _ops(), cuda_device
    monkeypatch.setattr(ops, "PAIR_FROM", pair_from)
    cached, new = [700, 0, 1111], [900, 129, 3]
    kvlens = [a + b for a, b in zip(cached, new)]
    rows, n_pages = _tables(kvlens, 2, 30)
    g = torch.Generator().manual_seed(31)
    kv = torch.randn((n_pages, nkv, 2, 16, hd), generator=g)
    for e, n in enumerate(kvlens):                # keys grow along the request
        for p in range((n + 15) // 16):
            kv[rows[e][p], :, 0] *= 0.2 + 3.0 * p * 16 / max(kvlens)
    rec = P.make_records(kv, kind)
    val = P.decode_records(rec, hd, kind)
    rec[rows[0][90], 0, 32 * hd + 5] = 255        # key 1445 of the first request
    T, qs = sum(new), [0, 900, 1029, 1032]
    q = torch.randn((T, nh * hd), generator=g).to(torch.bfloat16)
    per, scale = ops.prefill_quant_tokens(nh, nkv, hd), 1.0 / math.sqrt(hd)
    out = torch.full((T, nh * hd), 3.0, dtype=torch.bfloat16, device=dev)
    args = (rec.to(dev), kind, _i32(rows, dev), _i32(qs, dev), _i32(kvlens, dev), 0, 3, sum((n + per - 1) // per for n in new), nh, nkv, hd, scale, window)
    ops.attention_prefill_quant(q.to(dev), out, *args, _ws(dev))
    again = torch.empty_like(out)
    ops.attention_prefill_quant(q.to(dev), again, *args, _ws(dev))
    assert torch.equal(out.nan_to_num(nan=7.0), again.nan_to_num(nan=7.0))
    got = out.cpu().double()
    for e in range(3):
        for i in sorted({0, 1, new[e] - 1, new[e] // 2, *range(3, new[e], 41)}):
            pos, t = cached[e] + i, qs[e] + i
            row = got[t].view(nh, hd)
            if e == 0 and P.mask_lo(pos, window or 0) <= 1445 <= pos:
                assert torch.isnan(row[:nh // nkv]).all()
                continue
            want, mag = P.attend(q[t].view(nh, hd), val, rows[e], pos, scale, window or 0)
            room = want.abs() * 2.0 ** -8 * (1 + 2.0 ** -8) + mag * (2.0 ** -8 + 2.0 ** -14)
            assert ((row - want).abs() <= room).all(), (e, i, ((row - want).abs() / room.clamp(min=1e-300)).max())
    ops.check_status(dev)


# ---- together -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
def test_a_prompt_and_tokens_behind_it_as_captured_steps(cuda_device, kind):
    """Prompts are stored and attended over, then tokens one by one with the step replayed as a graph: every step against the definition, from the cache's own values."""
    ops, dev = _ops(), cuda_device
    nh, nkv, hd, E, width = 16, 2, 64, 3, 6
    prompts, steps = [30, 17, 48], 6
    rows, n_pages = _tables([width * 16] * E, 1, 15, width)
    inv = (1.0 / 10000.0 ** (torch.arange(hd // 2).double() / (hd // 2))).float().to(dev)
    cache = torch.zeros((n_pages, nkv, ops.kv_quant_record(hd)), dtype=torch.uint8, device=dev)
    tab, ws, scale, w = _i32(rows, dev), _ws(dev), 1.0 / math.sqrt(hd), (nh + 2 * nkv) * hd
    g = torch.Generator().manual_seed(16)
    T, qs = sum(prompts), [0, 30, 47, 95]
    qkv = torch.randn((T, w), generator=g).to(torch.bfloat16).to(dev)
    pos = _i32([i for n in prompts for i in range(n)], dev)
    ent = _i32([e for e, n in enumerate(prompts) for _ in range(n)], dev)
    q, out = torch.empty((T, nh * hd), dtype=torch.bfloat16, device=dev), torch.empty((T, nh * hd), dtype=torch.bfloat16, device=dev)
    per = ops.prefill_quant_tokens(nh, nkv, hd)
    ops.rope_store_quant(qkv, q, pos, ent, tab, cache, kind, nh, nkv, hd, hd, inv, 1.0)
    ops.attention_prefill_quant(q, out, cache, kind, tab, _i32(qs, dev), _i32(prompts, dev), 0, E, sum((n + per - 1) // per for n in prompts), nh, nkv, hd, scale, None, ws)
    val = P.decode_records(cache.cpu(), hd, kind)
    for e, n in enumerate(prompts):
        want, mag = P.attend(q[qs[e + 1] - 1].cpu().view(nh, hd), val, rows[e], n - 1, scale, 0)
        assert ((out[qs[e + 1] - 1].cpu().double().view(nh, hd) - want).abs() <= want.abs() * 2.0 ** -8 * (1 + 2.0 ** -8) + mag * (2.0 ** -8 + 2.0 ** -14)).all()
    step_in = torch.zeros((E, w), dtype=torch.bfloat16, device=dev)
    kvl, at, who = _i32(prompts, dev), _i32(prompts, dev), _i32([0, 1, 2], dev)
    q1, o1 = torch.empty((E, nh * hd), dtype=torch.bfloat16, device=dev), torch.empty((E, nh * hd), dtype=torch.bfloat16, device=dev)

    def step():
        ops.rope_store_quant(step_in, q1, at, who, tab, cache, kind, nh, nkv, hd, hd, inv, 1.0)
        ops.attention_decode_quant(q1, o1, cache, kind, tab, kvl, E, nh, nkv, hd, scale, None, width * 16, ws, cached_before=True)
    kvl += 1
    step()                                        # (workspaces are made outside the capture)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(steps):
        step_in.copy_(torch.randn((E, w), generator=g).to(torch.bfloat16).to(dev))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        val = P.decode_records(cache.cpu(), hd, kind)
        _decode_check(o1.cpu(), q1.cpu(), val, rows, kvl.cpu().tolist(), nh, hd, scale, 0)
        v = step_in[:, (nh + nkv) * hd:].cpu().double().view(E, nkv, hd)
        for e in range(E):
            p = int(at[e])
            assert torch.equal(val[rows[e][p // 16], :, 1, p % 16], P.encode(v[e], kind)[0])
        kvl += 1
        at += 1
    ops.check_status(dev)


def test_another_stream(cuda_device):
    """Kernels go to the current stream: the same results there, behind work of that stream."""
    ops, dev = _ops(), cuda_device
    nh, nkv, hd, n = 8, 2, 128, 500
    rows, n_pages = _tables([n], 0, 17)
    tab, kvl = _i32(rows, dev), _i32([n], dev)
    qkv = torch.randn((n, (nh + 2 * nkv) * hd), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(dev)
    pos, ent = _i32(list(range(n)), dev), _i32([0] * n, dev)

    def go():
        cache, ws = torch.zeros((n_pages, nkv, ops.kv_quant_record(hd)), dtype=torch.uint8, device=dev), _ws(dev)
        q, out, one = (torch.empty((n, nh * hd), dtype=torch.bfloat16, device=dev) for _ in range(3))
        ops.rope_store_quant(qkv, q, pos, ent, tab, cache, "fp8_e4m3", nh, nkv, hd, 0, None, 1.0)
        per = ops.prefill_quant_tokens(nh, nkv, hd)
        ops.attention_prefill_quant(q, out, cache, "fp8_e4m3", tab, _i32([0, n], dev), kvl, 0, 1, (n + per - 1) // per, nh, nkv, hd, 0.1, None, ws)
        ops.attention_decode_quant(q[-1:], one, cache, "fp8_e4m3", tab, kvl, 1, nh, nkv, hd, 0.1, None, n, ws)
        return out, one[:1].clone(), cache
    here = go()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = go()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(here, there))


# ---- calls that are odd but allowed ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("pair_from", [0, 1 << 30])
@pytest.mark.parametrize("window", [None, 20])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prompts_beside_requests_without_tokens(cuda_device, monkeypatch, pair_from, window, hd):
    """Entries that bring nothing, with keys or without, change no bit of the others'; a replayed call takes the lengths that it finds."""
    ops, dev = _ops(), cuda_device
    monkeypatch.setattr(ops, "PAIR_FROM", pair_from)
    nh, nkv = 6, 2
    per = ops.prefill_quant_tokens(nh, nkv, hd)

    def descriptors(cached, new, width):
        kvlens = [a + b for a, b in zip(cached, new)]
        qs = [0]
        for n in new:
            qs.append(qs[-1] + n)
        return kvlens, qs
    cached, new = [0, 33, 0, 100, 16, 0], [0, 0, 70, 41, 1, 0]
    kvlens, qs = descriptors(cached, new, 10)
    rows, n_pages = _tables(kvlens, 1, 3, width=10)
    rec, _ = _cache(n_pages, nkv, hd, "fp8_e4m3", 4, spread=0.5)
    cache = rec.to(dev)
    q = torch.randn((sum(new), nh * hd), generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).to(dev)

    def run(out, rows, qs, kvlens, tiles, rule, ws):
        ops.attention_prefill_quant(q, out, cache, "fp8_e4m3", rows, qs, kvlens, 0, kvlens.numel(), tiles, nh, nkv, hd, 0.1, window, ws, n_tiles_rule=rule)
    tiles = sum((n + per - 1) // per for n in new)
    full = torch.full_like(q, 3.0)
    run(full, _i32(rows, dev), _i32(qs, dev), _i32(kvlens, dev), tiles, tiles, _ws(dev))
    some = torch.full_like(q, 3.0)
    keep = [2, 3, 4]
    _, qs2 = descriptors([cached[e] for e in keep], [new[e] for e in keep], 10)
    run(some, _i32([rows[e] for e in keep], dev), _i32(qs2, dev), _i32([kvlens[e] for e in keep], dev), tiles, tiles, _ws(dev))
    assert torch.equal(full, some) and not (full == 3.0).all(1).any()

    # captured for these lengths, replayed for others whose tiles are no more
    ws, d_rows, d_qs, d_kv, out = _ws(dev), _i32(rows, dev), _i32(qs, dev), _i32(kvlens, dev), torch.full_like(q, 3.0)
    run(out, d_rows, d_qs, d_kv, tiles, tiles, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(out, d_rows, d_qs, d_kv, tiles, tiles, ws)
    for other in ([0, 0, 70, 41, 1, 0], [0, 0, 5, 1, 0, 0], [0, 0, 0, 0, 0, 0], [0, 0, 30, 41, 1, 0]):
        kvl, qs3 = descriptors(cached, other, 10)
        d_qs.copy_(_i32(qs3, dev)), d_kv.copy_(_i32(kvl, dev)), out.fill_(3.0)
        graph.replay()
        want = torch.full_like(q, 3.0)
        run(want, _i32(rows, dev), _i32(qs3, dev), _i32(kvl, dev), tiles, tiles, _ws(dev))
        assert torch.equal(out, want) and (out[sum(other):] == 3.0).all() and not (out[:sum(other)] == 3.0).all(1).any()
    ops.check_status(dev)


def test_two_captured_steps_that_share_a_workspace(cuda_device):
    """A long and a short step of single tokens, captured over one workspace and replayed in turn: each gives what it gives alone."""
    ops, dev = _ops(), cuda_device
    nh, nkv, hd = 16, 2, 64
    ws, steps = _ws(dev), []
    for i, kvlens in enumerate(([3000, 17, 1200], [300] * 5)):
        rows, n_pages = _tables(kvlens, 0, i)
        rec, _ = _cache(n_pages, nkv, hd, "int8", i + 2)
        q = torch.randn((len(kvlens), nh * hd), generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).to(dev)
        steps.append((q, torch.zeros_like(q), rec.to(dev), "int8", _i32(rows, dev), _i32(kvlens, dev), len(kvlens), nh, nkv, hd, 0.1, None, max(kvlens)))
    alone = []
    for a in steps:
        ops.attention_decode_quant(*a, ws)
        alone.append(a[1].clone())
    torch.cuda.synchronize()
    graphs = []
    for a in steps:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            ops.attention_decode_quant(*a, ws)
    for i in (0, 1, 0, 0, 1):
        steps[i][1].zero_()
        graphs[i].replay()
        assert torch.equal(steps[i][1], alone[i])
    ops.check_status(dev)


@pytest.mark.parametrize("blocks", [None, 0, -4])
@pytest.mark.parametrize("nh", [4, 12])
def test_decode_of_a_thousand_requests(cuda_device, monkeypatch, blocks, nh):
    """More requests than a warp's lanes count at a time, many without a key, next to long ones."""
    ops, dev = _ops(), cuda_device
    nkv, hd, n = 1, 64, 1000
    if blocks is not None:
        monkeypatch.setattr(ops, "_quant_blocks", lambda *a: blocks)
    g = torch.Generator().manual_seed(9)
    kvlens = [0 if i % 3 == 0 else int(torch.randint(1, 90, (1,), generator=g)) for i in range(n)]
    kvlens[500], kvlens[999] = 2500, 700
    rows, n_pages = _tables(kvlens, 0, 7)
    rec, val = _cache(n_pages, nkv, hd, "fp8_e4m3", 8)
    q = torch.randn((n, nh * hd), generator=g).to(torch.bfloat16)
    out = torch.full((n, nh * hd), 3.0, dtype=torch.bfloat16, device=dev)
    ops.attention_decode_quant(q.to(dev), out, rec.to(dev), "fp8_e4m3", _i32(rows, dev), _i32(kvlens, dev), n, nh, nkv, hd, 0.125, None, max(kvlens), _ws(dev))
    pick = sorted({0, 1, 2, 31, 32, 33, 499, 500, 501, 998, 999, *range(7, n, 61)})
    _decode_check(out.cpu()[pick], q[pick], val, [rows[e] for e in pick], [kvlens[e] for e in pick], nh, hd, 0.125, 0)
    assert not out.cpu()[::3][[i for i in range(334) if kvlens[3 * i] == 0]].any()
    ops.check_status(dev)


def test_store_of_many_tokens_is_the_store_of_few(cuda_device):
    """Warps a token are chosen by the number of tokens: the same codes and queries either way."""
    ops, dev = _ops(), cuda_device
    nh, nkv, hd, T = 8, 2, 128, 6000
    rows, n_pages = _tables([T], 0, 1)
    qkv = torch.randn((T, (nh + 2 * nkv) * hd), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(dev)
    pos, entry, tab = torch.arange(T, dtype=torch.int32, device=dev), torch.zeros(T, dtype=torch.int32, device=dev), _i32(rows, dev)
    freq = (10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)).float().to(dev)
    got = []
    for step in (T, 37):
        cache, q = torch.zeros((n_pages, nkv, 32 * hd + 32), dtype=torch.uint8, device=dev), torch.zeros((T, nh * hd), dtype=torch.bfloat16, device=dev)
        for a in range(0, T, step):
            b = min(T, a + step)
            ops.rope_store_quant(qkv[a:b], q[a:b], pos[a:b], entry[a:b], tab, cache, "int8", nh, nkv, hd, hd, freq, 1.0)
        got.append((cache, q))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
